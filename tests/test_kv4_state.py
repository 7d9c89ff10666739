"""What the 4-bit cache and its operators keep between calls, without a GPU: default workspaces under
capture and error bits."""
from __future__ import annotations

import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from mrun_b200 import _lib, paged_kv4

from test_paged_kv4 import _decode, _prefill


def test_a_captured_call_gets_memory_of_the_graphs_own(monkeypatch):
    """The stream's buffer is replaced by a larger one and serves eager calls: a graph must not hold it."""
    capturing = [False]
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    dev = torch.device("cpu", 0)
    for counters in (0, 64):
        scratch = _lib.StreamScratch()
        warm = scratch.get(dev, 1000, counters=counters)
        warm.fill_(1)
        capturing[0] = True
        first, second = (scratch.get(dev, 1000, counters=counters) for _ in range(2))
        capturing[0] = False
        eager = scratch.get(dev, 1000, counters=counters)
        assert eager.data_ptr() == warm.data_ptr()
        assert len({first.data_ptr(), second.data_ptr(), warm.data_ptr()}) == 3
        for buf in (first, second):
            assert buf.numel() >= 1000 and not buf[:counters or 1000].any()


def test_a_capture_on_a_stream_without_a_buffer(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    dev = torch.device("cpu", 0)
    scratch = _lib.StreamScratch()
    assert scratch.get(dev, 1000) is None  # callers that do without one
    buf = scratch.get(dev, 1000, counters=64)
    assert buf.numel() == 1000 and not buf[:64].any()
    assert scratch.get(dev, 0, counters=64) is None


def test_the_header_and_the_binding_agree_on_the_counters():
    header = (Path(__file__).resolve().parents[1] / "include" / "mrun_b200.h").read_text()
    assert int(re.search(r"#define MRB_KV4_COUNTER_BYTES (\d+)", header)[1]) == paged_kv4._COUNTER_BYTES


def _header() -> str:
    return (Path(__file__).resolve().parents[1] / "include" / "mrun_b200.h").read_text()


def test_every_error_bit_has_a_name_and_a_text():
    bits = {name: int(value) for name, value in re.findall(r"MRB_(KV_\w+) = (\d+),", _header())}
    assert bits and all(getattr(paged_kv4, name) == value for name, value in bits.items())
    assert sorted(paged_kv4._ERRORS) == sorted(bits.values())


def test_a_wait_that_ran_out_is_an_error():
    """A kernel whose bounded wait ran out has written what is no result: the cache says so."""
    cache = paged_kv4.PagedKV4Cache(num_layers=1, num_pages=2, kv_heads=1, head_dim=64, max_seqs=1,
                                    max_pages_per_seq=2, device=torch.device("cpu"))
    cache.error_flag.fill_(paged_kv4.KV_TIMEOUT)
    with pytest.raises(RuntimeError, match="ran out"):
        cache.check_errors()
    cache.check_errors()


def test_a_row_that_was_cut_is_an_error():
    cache = paged_kv4.PagedKV4Cache(num_layers=1, num_pages=2, kv_heads=1, head_dim=64, max_seqs=1,
                                    max_pages_per_seq=2, device=torch.device("cpu"))
    cache.error_flag.fill_(paged_kv4.KV_TOO_LONG)
    with pytest.raises(OverflowError, match="longer than"):
        cache.check_errors()


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_positions_that_cannot_be_rounded_up_are_refused(call):
    """2^31 - 16 tokens a row: their last step's end is past 32 bits."""
    pages = (2 ** 31 - 1) // 16
    assert call(_lib.load(), per=pages, stride=pages) == _lib.MRB_ERR_UNSUPPORTED


def test_reservations_of_a_4_bit_cache_hold_together():
    """Two sequences that were each promised room have it, against each other and against a prefill."""
    from mrun_b200.dense_engine import DenseDecoder

    dec = object.__new__(DenseDecoder)
    dec.kv_bits, dec.max_batch, dec.max_seq_len, dec.device = 4, 3, 256, torch.device("cpu")
    dec.kv = paged_kv4.PagedKV4Cache(num_layers=1, num_pages=6, kv_heads=1, head_dim=64, max_seqs=3,
                                     max_pages_per_seq=4, device=dec.device, page_size=64)
    dec.reserved = [0] * 3
    dec.kv.lengths[:] = torch.tensor([70, 0, 64])  # 2 + 0 + 1 pages
    dec.kv.free_count.fill_(3)
    dec.reserve(0, 192)  # one more page, which later calls may not take
    with pytest.raises(MemoryError):
        dec.reserve(1, 129)
    dec.reserve(1, 100)
    dec.reserve(0, 150)  # less than it has
    assert dec.reserved == [192, 100, 0]
    with pytest.raises(MemoryError):
        dec.reserve(2, 65)
    with pytest.raises(MemoryError):
        dec._room({2: 1})
    assert dec._room({0: 122, 1: 128}) == [70, 0]  # within their own
    with pytest.raises(MemoryError):
        dec._room({0: 123})
    with pytest.raises(OverflowError):
        dec.reserve(1, 257)
    dec.kv.release = lambda seqs: None
    dec.release(1)
    dec.reserve(2, 192)


def test_yarn_tables_take_every_key():
    """Published yarn configurations name a magnitude for all dimensions, and ramps between any two."""
    base = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    cpu = torch.device("cpu")

    def tables(**kw):
        return [t.double().numpy() for t in paged_kv4.scaled_rope_tables(64, 1e4, 7, cpu, scaling=base | kw)]

    plain = tables(attention_factor=1.0)
    for kw, mult in (({}, 0.1 * math.log(40) + 1), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
                     ({"mscale": 0.707, "mscale_all_dim": 1.0}, (0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1)),
                     ({"mscale": 0.707}, 0.1 * math.log(40) + 1),
                     ({"attention_factor": 2.0, "mscale": 0.7, "mscale_all_dim": 1.0}, 2.0)):
        for got, one in zip(tables(**kw), plain):
            assert np.allclose(got, mult * one, rtol=2 ** -22, atol=2 ** -22)

    def dim(turns):
        return 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(1e4))

    ramp = np.clip((np.arange(32) - dim(32)) / (dim(1) - dim(32)), 0, 1)
    inv = 1e4 ** -(np.arange(0, 64, 2) / 64)
    want = np.cos(np.arange(7)[:, None] * (inv * (1 - ramp) + inv / 40 * ramp))
    assert np.allclose(tables(truncate=False, attention_factor=1.0)[0], want, atol=2 ** -22)


@pytest.mark.parametrize("scaling", [{"rope_type": "spiral"}, {"rope_type": "linear"}, {"type": "yarn", "factor": 2.0},
                                     {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0}])
def test_rotary_scalings_that_are_not_whole_are_refused(scaling):
    with pytest.raises(ValueError):
        paged_kv4.scaled_rope_tables(16, 1e4, 4, torch.device("cpu"), scaling=scaling)
