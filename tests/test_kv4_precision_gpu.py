"""The attentions over the 4-bit cache against bounds from the roundings that each one makes.

With p the weights, s and m a group's scale and minimum and c its codes, to first order:

* an error d_t of token t's score moves an output by at most sum p_t d_t |v_t| + |o| sum p_t d_t
* decode: scores in fp32 of exact codes, d = 2^-19 scale sum |q| (|m| + 15 s) (sums of 128 terms and
  the subtraction of a maximum); weights times scales in fp16, 2^-11 sum p s c, and at least a quantum
  of 2^-25 relative to 2^7, for the largest product p s of any group: n 15 2^-32 max(p s)
* prefill: keys and values in fp16, d = 2^-11 scale sum |q k| and 2^-11 sum p |v|; weights in fp16,
  2^-11 sum p |v|; what is small beside its token, 2^-18 of the token's largest key or value
* both: fp32 sums 2^-18 sum p (|m| + 15 s), the output's rounding 2^-8 |o|"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_kv4_gpu import SHAPES, _bf, _i32

from oracle import kv4 as ok

pytestmark = pytest.mark.gpu


def _row(k, v, group, cuda, page=64):
    """One row of keys and values [n, hkv, d], cached: pool, table, and the oracle's view."""
    n, hkv, d = k.shape
    pages = -(-n // page)
    parts = []
    for x in (k, v):
        full = np.zeros((pages * page, hkv, d))
        full[:n] = x
        parts.append(ok.quantise(full.reshape(pages, page // 16, 16, hkv, d).transpose(0, 3, 1, 2, 4), group))
    pool = torch.from_numpy(ok.pack(*parts[0], *parts[1])).to(cuda)
    flat = tuple(tuple(np.moveaxis(x, 1, 3).reshape(pages * page, hkv, -1)[:n] for x in p) for p in parts)
    return pool, _i32([list(range(pages))], cuda), flat


def _bounds(q, cache, n, scale):
    """Output and bounds (decode's, prefill's) of one query [hq, d] over n tokens."""
    (kc, ks, km), (vc, vs, vm) = ((x[:n] for x in which) for which in cache)
    hq, d = q.shape
    k, v = ok.values(kc, ks, km), ok.values(vc, vs, vm)

    def wide(x):
        return np.repeat(x, d // x.shape[-1], -1)

    out, decode, prefill = (np.zeros((hq, d)) for _ in range(3))
    for h in range(hq):
        g = h // (hq // k.shape[1])
        aq = np.abs(q[h])
        score = k[:, g] @ q[h] * scale
        p = np.exp(score - score.max())
        p /= p.sum()
        out[h] = o = p @ v[:, g]
        av, step = np.abs(v[:, g]), wide(vs[:, g])
        both = 2.0 ** -8 * np.abs(o) + 2.0 ** -18 * (p @ (np.abs(wide(vm[:, g])) + 15 * step))

        def moved(e):
            return (p * e) @ av + np.abs(o) * (p @ e)

        exact = 2.0 ** -19 * abs(scale) * ((np.abs(wide(km[:, g])) + 15 * wide(ks[:, g])) @ aq)
        decode[h] = (both + moved(exact) + 2.0 ** -11 * (p @ (step * vc[:, g]))
                     + n * 15 * 2.0 ** -32 * (p * vs[:, g].max(-1)).max())
        small_k, small_v = (2.0 ** -18 * x.max(-1, keepdims=True) for x in (np.abs(k[:, g]), av))
        rounded = abs(scale) * ((2.0 ** -11 * np.abs(k[:, g]) + small_k) @ aq)
        prefill[h] = both + moved(exact + rounded) + p @ (2.0 ** -10 * av + small_v)
    return out, decode, prefill


def _check(k, v, q, group, cuda, scale=None, heads=None):
    """Both attentions of queries [1, hq, d] over one row, held to their bounds."""
    from mrun_b200.paged_kv4 import kv4_paged_attention, kv4_prefill_attention

    n, d = k.shape[0], k.shape[-1]
    pool, table, cache = _row(k, v, group, cuda)
    scale = d ** -0.5 if scale is None else scale
    common = dict(group=group, block_table=table, row_len=_i32([n], cuda), scale=scale)
    want, *bounds = _bounds(q[0], cache, n, scale)
    got = (kv4_paged_attention(_bf(q, cuda), pool, max_total_tokens=n, **common),
           kv4_prefill_attention(_bf(q, cuda), pool, q_starts=_i32([0, 1], cuda), **common))
    for name, x, bound in zip(("decode", "prefill"), got, bounds):
        err = np.abs(x[0].double().cpu().numpy() - want)
        assert (err <= bound).all(), (name, float((err / np.maximum(bound, 1e-300)).max()))  # (NaN fails too)


@pytest.mark.parametrize("head_dim,group", SHAPES)
@pytest.mark.parametrize("n", [1, 33, 700, 5000])
def test_ordinary_values(head_dim, group, n, cuda):
    rng = np.random.default_rng(n + head_dim + group)
    hq, hkv = 14, 2
    k, v = (ok.bf16(rng.standard_normal((n, hkv, head_dim)) + c * rng.standard_normal((hkv, head_dim))) for c in (1, 0))
    _check(k, v, ok.bf16(rng.standard_normal((1, hq, head_dim)) * 1.5), group, cuda)


@pytest.mark.parametrize("power", [8, 14, 20])
@pytest.mark.parametrize("head_dim,group", SHAPES)
def test_a_key_far_above_its_neighbours(head_dim, group, power, cuda):
    """A key 2^8 to 2^20 times as large as the others, which no query weighs: the others keep their bits."""
    rng = np.random.default_rng(power + head_dim + group)
    n, hq, hkv = 200, 8, 2
    k, v = (ok.bf16(rng.standard_normal((n, hkv, head_dim))) for _ in range(2))
    q = ok.bf16(rng.standard_normal((1, hq, head_dim)))
    q[..., 0] = np.abs(q[..., 0]) + 2  # all queries share a direction, which the key is against
    k[77] = 0
    k[77, :, 0] = -2.0 ** power
    _check(k, v, ok.bf16(q), group, cuda)


@pytest.mark.parametrize("power", [10, 14, 18])
@pytest.mark.parametrize("head_dim,group", [(64, 32), (128, 32), (128, 64)])
def test_value_groups_of_unlike_sizes(head_dim, group, power, cuda):
    """One group of dimensions whose values are 2^10 to 2^18 times as large as the others'."""
    rng = np.random.default_rng(power + head_dim + group)
    n, hq, hkv = 200, 8, 2
    k, v = (ok.bf16(rng.standard_normal((n, hkv, head_dim))) for _ in range(2))
    v[..., :group] *= 2.0 ** power
    _check(k, v, ok.bf16(rng.standard_normal((1, hq, head_dim))), group, cuda)


@pytest.mark.parametrize("scale", [1e-20, 1e-37, -1e-20, 0.0])
@pytest.mark.parametrize("n", [5, 64, 77])
def test_scales_that_vanish(scale, n, cuda):
    """Queries of zeros and a scale near the end of fp32: all tokens weigh alike."""
    rng = np.random.default_rng(n)
    k, v = (ok.bf16(rng.standard_normal((n, 2, 64))) for _ in range(2))
    q = ok.bf16(rng.standard_normal((1, 4, 64)))
    q[:, ::2] = 0
    _check(k, v, q, 32, cuda, scale=scale)
