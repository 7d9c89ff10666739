"""Every cached token counts once, however an attention's work is cut and joined.

Queries of zeros weigh the n tokens of a row alike, so an output is sum_t v_t / n. A row's tokens are
divided into windows, and a value is n in its window and zero elsewhere: the output is the
window's count. Once the values are minima (scale 0), the same in all dimensions, and once codes (minimum
0, scale n, code 1 or 0), with a window for each dimension, so that few passes visit every token. n is
rounded to bf16, so both are held exactly.

Weights of equal scores are equal powers of two and the sums whole numbers below 2^24, so what is left
is the division and the rounding to bf16, 2^-9 of the value, and in decode, where weights times scales
go to fp16 relative to a maximum that is no power of two, 2^-11: 2^-8 holds all of them. A token lost
or counted twice in a window of w tokens is off by 1 / w, so windows are at most 64 tokens wide."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_kv4_gpu import _i32

from oracle import kv4 as ok

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -8


class Marked:
    """A pool whose values are marked by windows of ``width`` tokens; its keys hold anything."""

    def __init__(self, lengths, hkv, head_dim, group, width, dev, seed=0):
        rng = np.random.default_rng(seed)
        self.lengths, self.hkv, self.d, self.ng, self.page, self.width = lengths, hkv, head_dim, head_dim // group, 64, width
        need = [-(-n // self.page) for n in lengths]
        self.pages = sum(need) + 1
        order = rng.permutation(self.pages).tolist()
        table = np.full((len(lengths), max(need + [1])), -1)
        at = np.full((self.pages, self.page), -1)  # what each place holds: a position, or nothing
        n = np.zeros((self.pages, 1))
        for r, count in enumerate(need):
            table[r, :count] = [order.pop() for _ in range(count)]
            where = np.arange(count * self.page).reshape(count, self.page)
            at[table[r, :count]] = np.where(where < lengths[r], where, -1)
            n[table[r, :count]] = lengths[r]
        self.table = _i32(table.tolist(), dev)
        self.at = torch.from_numpy(at).to(dev)
        self.held = torch.from_numpy(n).to(dev).to(torch.bfloat16).double()  # n of the row, as bf16
        self.windows = -(-max(lengths) // width)
        block = ok.block_bytes(head_dim, group)
        self.pool = torch.from_numpy(rng.integers(0, 256, (self.pages, hkv, self.page // 16, block), dtype=np.uint8)).to(dev)
        half, par = 8 * head_dim, 64 * self.ng
        self.codes, self.params = self.pool[..., half:2 * half], self.pool[..., 2 * half + par:]
        keys = torch.tensor([0.25, -1.5], dtype=torch.bfloat16, device=dev).repeat(16 * self.ng)
        self.pool[..., 2 * half:2 * half + par] = keys.view(torch.uint8)

    def _set(self, codes, scale, minimum):
        """Of each place: codes [pages, page, d], scale and minimum [pages, page]."""
        packed = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8).view(self.pages, self.page // 16, -1)
        pair = torch.stack([scale, minimum], -1).to(torch.bfloat16)[:, :, None].expand(-1, -1, self.ng, -1)
        pair = pair.reshape(self.pages, self.page // 16, -1).view(torch.uint8)
        for part, value in ((self.codes, packed), (self.params, pair)):
            part.copy_(value[:, None].expand(-1, self.hkv, -1, -1))

    def passes(self):
        """Sets the marks, pass after pass: the window of each dimension."""
        window = torch.where(self.at >= 0, self.at // self.width, -1)
        zero = torch.zeros_like(self.at)
        for w in range(0, self.windows, max(1, self.windows // 24)):
            self._set(zero[..., None].expand(-1, -1, self.d) + 9, zero, torch.where(window == w, self.held, 0.0))
            yield torch.full((self.d,), w, device=self.at.device)
        for w in range(0, self.windows, self.d):
            mine = w + torch.arange(self.d, device=self.at.device)
            self._set((window[..., None] == mine).int(), self.held.expand_as(self.at), zero)
            yield mine

    def want(self, row, sees, windows):
        """Outputs [queries, d] of queries of the given rows that see that many tokens."""
        n = torch.tensor(self.lengths, device=row.device).to(torch.bfloat16).double()[row]
        count = (sees[:, None] - windows * self.width).clamp(0, self.width)
        return n[:, None] * count / sees[:, None].clamp(min=1)


def _close(out, want, what):
    """out [queries, heads, d] equal to ``want`` [queries, d] within TOL."""
    want = want[:, None]
    far = (out.double() - want).abs()
    bad = far > TOL * want.abs()
    assert not bad.any(), (what, int(bad.sum()), float(far.max()))


@pytest.mark.parametrize("lengths,hq,hkv,head_dim,group,width", [
    ([9005], 28, 4, 128, 128, 64),              # few groups: equal parts, one a CTA
    ([40000], 16, 1, 128, 64, 64),              # one group in more parts than are joined in one go
    ([30000, 17, 12345], 2, 1, 64, 32, 64),
    ([4096, 1, 0, 777, 2049, 31, 33, 4000], 32, 4, 128, 128, 64),
    ([300, 0, 517] * 30 + [4097], 32, 8, 128, 32, 61),   # many groups: ranges cut anywhere
    ([90, 64, 0, 33, 1] * 140, 8, 4, 64, 64, 32),        # more rows than a launch takes
])
def test_decode_counts_every_token_once(lengths, hq, hkv, head_dim, group, width, cuda):
    from mrun_b200.paged_kv4 import kv4_paged_attention

    m = Marked(lengths, hkv, head_dim, group, width, cuda, seed=len(lengths))
    q = torch.zeros(len(lengths), hq, head_dim, dtype=torch.bfloat16, device=cuda)
    sees = torch.tensor(lengths, device=cuda)
    for windows in m.passes():
        out = kv4_paged_attention(q, m.pool, group=group, block_table=m.table, row_len=sees.int(),
                                  max_total_tokens=max(lengths))
        _close(out, m.want(torch.arange(len(lengths), device=cuda), sees, windows), windows[:2])


@pytest.mark.parametrize("new,ctx,hq,hkv,head_dim,group,width", [
    ([5], [9000], 28, 4, 128, 128, 64),                    # few tiles, each in many parts
    ([1, 2], [20000, 3], 8, 8, 64, 32, 64),
    ([40, 1, 300], [6000, 11000, 0], 16, 1, 128, 64, 64),  # long and short tiles in one line
    ([1 + i % 3 for i in range(700)], [i % 50 for i in range(700)], 8, 8, 64, 64, 1),  # many pieces a CTA
    ([1] * 400 + [260], [0] * 400 + [3000], 12, 2, 128, 32, 64),
    ([4096], [0], 28, 4, 128, 128, 64),
    ([700], [16000], 4, 1, 64, 64, 64),
])
def test_prefill_counts_every_token_once(new, ctx, hq, hkv, head_dim, group, width, cuda):
    from mrun_b200.paged_kv4 import kv4_prefill_attention

    lengths = [a + b for a, b in zip(new, ctx)]
    m = Marked(lengths, hkv, head_dim, group, width, cuda, seed=len(new) + 7)
    starts = [0, *np.cumsum(new).tolist()]
    q = torch.zeros(starts[-1], hq, head_dim, dtype=torch.bfloat16, device=cuda)
    row = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(cuda)
    sees = torch.arange(1, starts[-1] + 1, device=cuda) + (torch.tensor(ctx) - torch.tensor(starts[:-1])).to(cuda)[row]
    for windows in m.passes():
        out = kv4_prefill_attention(q, m.pool, group=group, block_table=m.table, q_starts=_i32(starts, cuda),
                                    row_len=_i32(lengths, cuda))
        _close(out, m.want(row, sees, windows), windows[:2])
