"""Attention of rows that share a prefix right behind the kernels that append their keys, as a decoder's step has it: what those write has to be there."""
import pytest
import torch

from ironpangu_b200.ops import decode as K
from ironpangu_b200.ops import shared_prefix as S

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("rows,heads,kv,dim,shared", [(12, 8, 2, 64, 500), (24, 32, 8, 128, 4001), (204, 8, 2, 128, 700), (600, 8, 2, 64, 300), (150, 32, 8, 128, 2000)])
def test_behind_the_append(rows, heads, kv, dim, shared):
    """Parts and merge; the prefix by tiles ahead of them; four warps a row; one. Steps in one graph against steps that are waited for one by one, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    page, steps, own = 16, 6, 40
    front, each = shared // page, -(-(shared + own) // page) - shared // page
    tables = [list(range(front + 1)) + [-1] * (each - 1)] + [list(range(front)) + list(range(front + 1 + i * each, front + 1 + (i + 1) * each)) for i in range(rows)]
    table = torch.tensor(tables, dtype=I32, device="cuda")
    pages = front + 1 + rows * each
    caches = [torch.randn(pages, page, kv, dim, generator=g, device="cuda").to(BF16) for _ in range(2)]
    rows_in = torch.randn(steps, rows, (heads + 2 * kv) * dim, generator=g, device="cuda").to(BF16)
    first = shared + torch.randint(0, own - steps, (rows,), generator=g, device="cuda")
    groups = torch.tensor([[0, rows, shared, 0]], dtype=I32, device="cuda")
    slots = torch.arange(1, rows + 1, dtype=I32, device="cuda")
    status = torch.zeros(1, dtype=I32, device="cuda")
    scratch = torch.empty(S.scratch_bytes(rows, heads, kv, dim), dtype=torch.uint8, device="cuda")
    k, v, qkv, positions = caches[0].clone(), caches[1].clone(), torch.empty_like(rows_in[0]), torch.empty(rows, dtype=I32, device="cuda")
    out = torch.empty(steps, rows, heads * dim, dtype=BF16, device="cuda")

    def step(i, wait):
        positions.copy_(first + i)
        qkv.copy_(rows_in[i])
        wait()
        K.gqa_rope_kv_write(qkv, positions, slots, table, k, v, heads=heads, kv_heads=kv, head_dim=dim, status_ptr=status.data_ptr())
        wait()
        S.attention(qkv, k, v, positions, slots, table, groups, heads=heads, kv_heads=kv, head_dim=dim, scale=dim ** -0.5, scratch=scratch, out=out[i], status_ptr=status.data_ptr())
        wait()

    for i in range(steps):
        step(i, torch.cuda.synchronize)
    want, want_k = out.clone(), k.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.copy_(caches[0])
        v.copy_(caches[1])
        for i in range(steps):
            step(i, lambda: None)
    for again in range(10):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(k, want_k) and torch.equal(out, want), again
    assert int(status) == 0 and bool(want.isfinite().all())


@gpu
@pytest.mark.parametrize("rows,length", [(205, 500), (600, 130)])
def test_a_decoder_with_many_continuations(rows, length):
    """The last layer's attention of every step against the definition in 64 bits, from the step's own queries and caches."""
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric
    from ironpangu_b200.runtime.continuations import Continuations

    cfg = G.DenseConfig.tiny(2)
    dec = G.DenseDecoder(cfg, G.shard_weights(cfg, G.random_full_weights(cfg, 3), 0, 1, "cuda"), Fabric(0, 1), max_tokens=rows, max_context=length + 30, num_slots=rows + 1, keep_logits=True,
                         page_pool=True)
    c = Continuations(dec, shared_prefix=True)
    prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
    c.start(prompt, rows, temperature=1.5, top_k=0, seed=3)
    hd, per = cfg.head_dim, dec.hq // dec.hk
    for _ in range(20):                            # the first one is run, the others are replayed
        before = dec.positions.clone()
        c.step()
        for t in (0, 1, 2, 3, rows // 2, rows - 1):
            at = torch.arange(int(before[t]) + 1, device="cuda")
            pages = dec.page_table[int(dec.slots[t])].long()[at // cfg.page_tokens]
            k, v = (x[-1][pages, at % cfg.page_tokens].to(F64).repeat_interleave(per, 1) for x in (dec.k_cache, dec.v_cache))
            w = torch.softmax(torch.einsum("hd,jhd->hj", dec.qkv[t, :dec.hq * hd].view(dec.hq, hd).to(F64), k) / hd ** 0.5, 1)
            want = torch.einsum("hj,jhd->hd", w, v).reshape(-1)
            # rounded once; 15-bit weights of f32 scores
            room = want.abs() * 2 ** -8 + torch.einsum("hj,jhd->hd", w, v.abs()).reshape(-1) * 2 ** -14
            assert bool(((dec.attn[t].to(F64) - want).abs() <= room).all())
    c.check()
    c.end()
