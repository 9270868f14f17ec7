"""Several continuations of one prompt on one GPU: the prompt runs once, its pages are shared by as many sequence slots as continuations are wanted, and a decode step
of all of them - pages taken, layers, sampling, the sampled tokens fed back - is one CUDA graph without the host. Continuations can be drawn again with repeats
(:meth:`Continuations.resample`: those that were not drawn end, those drawn twice go on separately, as particles and beams do), set aside in a second pool and packed.

The decoder is a ``models.dense_gqa.DenseDecoder`` with ``page_pool`` and ``keep_logits``, bf16 or 4-bit weights; slot 0 holds the prompt and slot 1 + i continuation i."""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from ..ops import decode as K
from ..ops import pages as P

I32 = torch.int32


class Continuations:
    def __init__(self, decoder, *, prefill=None, store_pages: int = 0):
        """``prefill``: a ``models.dense_prefill.DensePrefill`` of the decoder; without one the prompt goes through the decode kernels. ``store_pages``: pages of the second
        pool that :meth:`set_aside` copies to."""
        if decoder.pool is None or decoder.logits is None:
            raise ValueError("continuations need a decoder with page_pool and keep_logits")
        self.dec, self.prefill, self.pool = decoder, prefill, decoder.pool
        self.width = min(decoder.T, decoder.num_slots - 1)
        dev = decoder.tokens.device
        i32 = lambda v: torch.tensor(v, dtype=I32, device=dev)
        self._first, self._children, self._lengths = i32([0]), i32(list(range(1, self.width + 1))), torch.zeros(self.width, dtype=I32, device=dev)
        self._tokens = torch.zeros(1, dtype=I32, device=dev)
        self.seeds, self.counters = torch.zeros(self.width, dtype=torch.int64, device=dev), torch.zeros(self.width, dtype=torch.int64, device=dev)
        self.inv_temp, self.top_p = torch.ones(self.width, device=dev), torch.ones(self.width, device=dev)
        self.ids = torch.zeros(self.width, dtype=I32, device=dev)
        self._scratch = torch.empty(self.width * ((decoder.logits.shape[1] + 4095) // 4096) * 128, dtype=torch.float32, device=dev)
        self._graphs = {}
        self.n = self.length = 0              # continuations, positions of each
        self.store = [torch.empty(store_pages, *c.shape[1:], dtype=c.dtype, device=dev) for c in decoder.k_cache + decoder.v_cache] if store_pages else []
        self._store = P.PageSet(self.store) if store_pages else None
        self._store_free = list(range(store_pages))[::-1]
        self._aside = {}                      # continuations that were set aside: their pages in the second pool
        self._ran = self._broken = False      # there was a run, whose reports may still lie in the status words; the continuations are not what their tokens say

    # -- prompt --------------------------------------------------------------------------------------------------------------
    def start(self, prompt: Sequence[int], n: int, *, temperature: float = 1.0, top_k: int = 50, top_p: float = 1.0, seed: int = 0) -> torch.Tensor:
        """Runs the prompt, forks it ``n`` times and samples the first token of each continuation (device tensor ``[n]``). ``temperature`` 0: greedy. Continuations that were
        there are ended first, and nothing that :meth:`check` would have said about them is said any more. Where this raises there are none."""
        d = self.dec
        if not 1 <= n <= self.width:
            raise ValueError(f"{n} continuations: this decoder takes 1 to {self.width}")
        if not 1 <= len(prompt) <= d.max_context:
            raise ValueError(f"a prompt of {len(prompt)} tokens in a context of {d.max_context}")
        if not 1 <= top_k <= 64:
            raise ValueError(f"top_k of {top_k}: 1 to 64")
        self.end()
        if self._ran:
            self.pool.status.zero_()
            if d.fabric.status():             # (waits for the kernels that may still set it)
                d.fabric.clear_status()
        self._ran = True
        try:
            self._begin(prompt, n, temperature, top_k, top_p, seed)
            self.check()
        except BaseException:
            self._release()
            raise
        self.n, self.length = n, len(prompt)
        return self.ids[:n]

    def _begin(self, prompt: Sequence[int], n: int, temperature: float, top_k: int, top_p: float, seed: int) -> None:
        d = self.dec
        self.top_k = 1 if temperature <= 0 else top_k
        self.inv_temp[:n].fill_(1e4 if temperature <= 0 else 1.0 / temperature)
        self.top_p[:n].fill_(1.0 if temperature <= 0 else top_p)
        first = (seed * 0x9E3779B1 + (1 << 63)) % (1 << 64) - (1 << 63)      # of 64 bits, as any seed is
        self.seeds[:n].copy_(torch.arange(n, dtype=torch.int64) + first)
        self.counters.zero_()
        self._tokens.fill_(len(prompt))
        self.pool.extend(self._first, self._tokens)
        self.pool.check()
        tokens = torch.tensor(list(prompt), dtype=I32, device=d.tokens.device)
        step = self.prefill.M if self.prefill is not None else d.T
        for p in range(0, len(prompt), step):
            part = tokens[p:p + step]
            if self.prefill is not None:
                self.prefill.forward(part, p, 0)
                last = 0
            else:
                m = part.numel()
                d.tokens[:m].copy_(part)
                d.positions[:m].copy_(torch.arange(p, p + m, dtype=I32))
                d.slots[:m].zero_()
                d.forward(m)
                last = m - 1
        self.pool.fork(self._first.expand(n).contiguous(), self._children[:n])
        if last:
            d.logits[0].copy_(d.logits[last])
        if n > 1:
            d.logits[1:n].copy_(d.logits[:1].expand(n - 1, -1))
        self._sample(n)
        d.positions[:n].fill_(len(prompt))
        d.slots[:n].copy_(self._children[:n])

    def _sample(self, n: int) -> None:
        d = self.dec
        for t in range(0, n, 64):             # the sampling kernel takes 64 rows
            e = min(n, t + 64)
            K.sample_topk(d.logits[t:e], d.fabric, top_k=self.top_k, inv_temperature=self.inv_temp[t:e], top_p=self.top_p[t:e], seeds=self.seeds[t:e],
                          counters=self.counters[t:e], scratch=self._scratch, out_ids=self.ids[t:e])
        d.tokens[:n].copy_(self.ids[:n])

    # -- steps ---------------------------------------------------------------------------------------------------------------
    def _step(self, n: int) -> None:
        d = self.dec
        torch.add(d.positions[:n], 1, out=self._lengths[:n])
        self.pool.extend(self._children[:n], self._lengths[:n])
        d.forward(n)
        self._sample(n)
        d.positions[:n].add_(1)

    def step(self) -> torch.Tensor:
        """The next token of every continuation (device tensor ``[n]``): one graph replay. A pool that has run out of pages shows in :meth:`check`, and the tokens since the check
        before it are not to be used then."""
        self._all_here()
        if self.length >= self.dec.max_context:
            raise OverflowError("the continuations run past the context")
        self.length += 1
        key = (self.n, self.top_k)
        g = self._graphs.get(key)
        if g is not None:
            g.replay()
        else:
            self._step(self.n)                # the real run of this step (and the warm-up of the capture)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):         # records only
                self._step(self.n)
            self._graphs[key] = g
        return self.ids[:self.n]

    def _all_here(self) -> None:
        self._sound()
        if self._aside:
            raise RuntimeError(f"continuations {sorted(self._aside)} are set aside: take_up() first")

    def _sound(self) -> None:
        if not self.n:
            raise RuntimeError("no continuations: start() first")
        if self._broken:
            raise RuntimeError("a step was refused: the continuations have to be ended")

    def check(self) -> None:
        """Raises IndexError when a resampling named a parent out of range (nothing was resampled then), OverflowError when a step or a resampling found too few free pages,
        RuntimeError when a kernel gave up or met an index out of range. After the latter two the continuations are not what their tokens say - positions whose keys and values
        were never written - and nothing but :meth:`end` and :meth:`start` takes them (waits for the device)."""
        if self._broken:
            self._sound()
        lacked, word = int(self.pool.status) & P.NO_PAGES, self.dec.fabric.status()
        self._broken = bool(lacked or word)
        if word:
            self.dec.fabric.clear_status()
        self.pool.check()                     # (pages that lacked are what kernels reported as out of range)
        if word:
            raise RuntimeError(f"continuations: kernel status word = {word}")

    def resample(self, parents: torch.Tensor) -> None:
        """Continuation ``i`` goes on from what ``parents[i]`` is now (int32 ``[n]`` on the device, out of 0 .. n - 1, with repeats). What is refused shows in :meth:`check`."""
        self._all_here()
        n = self.n
        if parents.shape != (n,) or parents.dtype != I32:
            raise ValueError(f"parents must be int32 [{n}]")
        inside = (parents >= 0) & (parents < n)
        self.pool.fork(torch.where(inside, parents + 1, -1), self._children[:n])
        now = self.dec.tokens[:n]
        now.copy_(torch.where(inside.all(), now.index_select(0, parents.long().clamp(0, n - 1)), now))

    def end(self) -> None:
        """Gives back all pages, those that were set aside among them."""
        if self.n:
            self._release()

    def _release(self) -> None:
        self.pool.free(self._children)
        self.pool.free(self._first)
        for ids in self._aside.values():
            self._store_free += ids.tolist()
        self._aside = {}
        self._broken = False
        self.n = self.length = 0

    # -- setting aside ---------------------------------------------------------------------------------------------------------
    def set_aside(self, i: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Copies continuation ``i`` to the second pool and gives its pages back; :meth:`take_up` brings it back from what this returns, and no step can be taken before."""
        if not 0 <= i < self.n or i in self._aside:
            raise ValueError(f"no continuation {i}")
        self._sound()
        length = int(self.pool.lengths[1 + i])
        if length != self.length:             # a step was refused
            self.check()
            raise RuntimeError(f"continuation {i} holds {length} positions of {self.length}")
        count = -(-length // self.pool.page_tokens)
        if count > len(self._store_free):
            raise OverflowError(f"{count} pages to set aside, {len(self._store_free)} free")
        dev = self._tokens.device
        ids = torch.tensor([self._store_free.pop() for _ in range(count)], dtype=I32, device=dev)
        rows = (length - self.pool.page_tokens * torch.arange(count, device=dev)).clamp(max=self.pool.page_tokens).to(I32)
        P.copy(self.pool.pages, self._store, self.pool.table[1 + i, :count], ids, rows)
        self.pool.free(self._children[i:i + 1])
        self._aside[i] = ids
        return ids, rows

    def take_up(self, i: int, held: Tuple[torch.Tensor, torch.Tensor]) -> None:
        """Continuation ``i``, which was set aside, has its pages again. OverflowError where pages lack: nothing has changed then, and it can be asked for again."""
        ids, rows = held
        if self._aside.get(i) is not ids:
            raise ValueError(f"this is not what continuation {i} was set aside as")
        self.check()
        count = ids.numel()
        length = (count - 1) * self.pool.page_tokens + rows[-1:] if count else torch.zeros(1, dtype=I32, device=ids.device)
        self.pool.extend(self._children[i:i + 1], length.to(I32))
        self.pool.check()
        P.copy(self._store, self.pool.pages, ids, self.pool.table[1 + i, :count], rows)
        del self._aside[i]
        self._store_free += ids.tolist()

    def pack(self) -> int:
        """Live pages into the lowest places; returns their number."""
        self.pool.compact()
        return int(self.pool.live)

    def generate(self, prompt: Sequence[int], n: int, max_new_tokens: int, eos: int = -1, **sampling) -> List[List[int]]:
        """``n`` continuations of up to ``max_new_tokens`` tokens, each cut off behind its first ``eos``. Ended also where this raises."""
        if max_new_tokens < 1:
            raise ValueError(f"{max_new_tokens} tokens: at least one")
        first = self.start(prompt, n, **sampling)
        try:
            steps = [first.clone()]
            for _ in range(max_new_tokens - 1):
                steps.append(self.step().clone())
            self.check()
            rows = torch.stack(steps, 1).tolist()
        finally:
            self.end()
        return [r[:r.index(eos) + 1] if eos in r else r for r in rows]
