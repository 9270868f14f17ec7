"""The worker's --weights-int4 and the runtime option behind it: where it is taken, where it is refused, and that what it serves is the decoder with 4-bit weights."""
import sys

import pytest

from ironpangu_b200.runtime.options import RuntimeOptions


def test_the_option_by_name_and_environment():
    assert RuntimeOptions().weights_int4 is False
    for o in (RuntimeOptions.from_env({"IFAB_WEIGHTS_INT4": "1"}), RuntimeOptions.from_env({}, ["weights_int4=on"]), RuntimeOptions.from_env({"IFAB_WEIGHTS_INT4": "0"}, ["weights-int4=1"])):
        assert o.weights_int4 is True and o.changed() == {"weights_int4": True}


@pytest.mark.parametrize("argv", [["--model", "tiny", "--weights-int4"], ["--model", "hybrid-tiny", "--set", "weights_int4=1"], ["--bundle", "/nowhere", "--model", "dense-tiny", "--weights-int4"]])
def test_models_without_4_bit_linears_refuse_it(argv, monkeypatch):
    from ironpangu_b200.runtime import engine_worker

    monkeypatch.setattr(sys, "argv", ["engine_worker", *argv])
    with pytest.raises(SystemExit, match="has no 4-bit linears"):
        engine_worker.main()


@pytest.mark.gpu
@pytest.mark.parametrize("options", ["--weights-int4", "--executor model --set weights_int4=1"])
def test_the_worker_serves_4_bit_weights(options):
    """Server, socket, worker, kernels: the tokens of the decoder whose weights were quantised here from the same matrices."""
    import torch

    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric
    from test_server import Server

    s = Server("--spawn", f"{sys.executable} -m ironpangu_b200.runtime.engine_worker --model dense-tiny --max-num-seqs 3 --max-model-len 128 --greedy-only {options}",
               "--accept-seconds", "300", timeout=400)
    try:
        cfg, fab = G.DenseConfig.tiny(2), Fabric(0, 1)
        weights = G.quantise_weights(G.random_rank_weights(cfg, 0, 1, torch.device("cuda", 0), seed=0))
        dec = G.DenseDecoder(cfg, weights, fab, max_tokens=8, max_context=128)
        for prompt in ([5, 77, 300, 12, 999, 41, 8, 650, 3, 17, 256], [9]):
            status, got = s.post("/inference/v1/generate", {"token_ids": prompt, "sampling_params": {"max_tokens": 6}}, timeout=120)
            assert status == 200, got
            row, want = list(prompt), []
            for p in range(len(prompt) + 5):
                dec.tokens[:1].fill_(row[p])
                dec.positions[:1].fill_(p)
                dec.slots[:1].zero_()
                token = int(dec.forward(1)[0])
                if p >= len(prompt) - 1:
                    want.append(token)
                    row.append(token)
            assert got["token_ids"] == want
        fab.close()
    finally:
        s.close()
