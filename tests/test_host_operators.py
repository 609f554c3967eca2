"""Argument checks, workspace sizes and registration of the window, shared-prefix and beam operators (no GPU).

The refused calls pass small integers where device pointers would stand: nothing may touch them.
"""

import ctypes

import pytest
import torch

from femtovllm_b200 import capi, ops

INVALID, UNSUPPORTED, MISALIGNED = 1, 2, 3
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def _status(lib, name):
    return next(i for i in range(32) if lib.fvb_status_string(i) == name.encode())


def _call(fn, base, over):
    a = dict(base)
    unknown = set(over) - set(a)
    assert not unknown
    a.update(over)
    return fn(*a.values())


ATTENTION = dict(q=16, q_ts=128, q_hs=256, out=16, o_ts=128, o_hs=256, k=16, v=16, num_blocks=10, hq=8, hkv=2, d=128,
                 page=16)
DECODE = dict(ATTENTION, b=2, tables=16, columns=4, lens=16, max_kv=50, window=20, sinks=4, dtype=1, ws=256, ws_bytes=BIG,
              stream=None)
PREFILL = dict(ATTENTION, b=2, tokens=5, cu=16, max_q=3, tables=16, columns=4, lens=16, positions=16, window=20, sinks=4,
               dtype=1, ws=256, ws_bytes=BIG, stream=None)
SHARED = dict(ATTENTION, b=2, tables=16, columns=4, lens=16, max_kv=50, cu_groups=16, groups=1, prefix=16, max_prefix=32,
              dtype=1, ws=256, ws_bytes=BIG, stream=None)

COMMON = [
    (dict(d=96), UNSUPPORTED),
    (dict(hq=7), UNSUPPORTED),
    (dict(page=32), UNSUPPORTED),
    (dict(dtype=7), UNSUPPORTED),
    (dict(q=8), MISALIGNED),
    (dict(q_ts=129), MISALIGNED),
    (dict(o_hs=-8), INVALID),
    (dict(num_blocks=0), INVALID),
    (dict(num_blocks=1 << 30), UNSUPPORTED),
    (dict(b=-1), INVALID),
    (dict(lens=None), INVALID),
    (dict(ws=128), MISALIGNED),
]


@pytest.mark.parametrize("over,status", COMMON + [
    (dict(window=0), INVALID),
    (dict(window=-5), INVALID),
    (dict(sinks=-1), INVALID),
    (dict(max_kv=65), INVALID),  # past the table row
    (dict(max_kv=-1), INVALID),
    (dict(b=70000, max_kv=1), UNSUPPORTED),
])
def test_window_decode_refuses(lib, over, status):
    assert _call(lib.fvb_paged_attention_window_decode, DECODE, over) == status


@pytest.mark.parametrize("over,status", COMMON + [
    (dict(window=0), INVALID),
    (dict(sinks=-1), INVALID),
    (dict(cu=None), INVALID),
    (dict(positions=None), INVALID),
    (dict(tokens=-1), INVALID),
    (dict(max_q=-1), INVALID),
    (dict(tokens=1 << 31), UNSUPPORTED),
])
def test_window_prefill_refuses(lib, over, status):
    assert _call(lib.fvb_paged_attention_window_prefill, PREFILL, over) == status


@pytest.mark.parametrize("over,status", COMMON + [
    (dict(groups=-1), INVALID),
    (dict(cu_groups=None), INVALID),
    (dict(prefix=None), INVALID),
    (dict(max_prefix=-16), INVALID),
    (dict(max_kv=65), INVALID),
    (dict(groups=70000), UNSUPPORTED),
])
def test_shared_prefix_refuses(lib, over, status):
    assert _call(lib.fvb_paged_attention_shared_prefix_decode, SHARED, over) == status


def test_no_work_returns_before_the_workspace_is_looked_at(lib):
    assert _call(lib.fvb_paged_attention_window_decode, DECODE, dict(b=0, ws=None, ws_bytes=0)) == 0
    assert _call(lib.fvb_paged_attention_window_prefill, PREFILL, dict(b=0, tokens=0, ws=None, ws_bytes=0)) == 0
    assert _call(lib.fvb_paged_attention_shared_prefix_decode, SHARED, dict(b=0, ws=None, ws_bytes=0)) == 0
    assert _call(lib.fvb_beam_search_select, SELECT, dict(requests=0, ws=None, ws_bytes=0)) == 0
    assert _call(lib.fvb_beam_reorder_kvcache, _reorder(), dict(requests=0)) == 0


def test_small_workspaces_are_refused(lib):
    small = _status(lib, "FVB_ERR_WORKSPACE_TOO_SMALL")
    long = dict(columns=4096, max_kv=65536, max_prefix=60000)
    for dtype in (0, 1):
        need = lib.fvb_paged_attention_shared_prefix_workspace_size(2, 8, 2, 128, 65536, 1, 60000, dtype)
        assert need > 0
        assert _call(lib.fvb_paged_attention_shared_prefix_decode, SHARED,
                     dict(long, dtype=dtype, q_ts=256, q_hs=512, ws_bytes=need - 1)) == small
        assert _call(lib.fvb_paged_attention_shared_prefix_decode, SHARED, dict(long, dtype=dtype, ws=None)) == small
    need = lib.fvb_beam_search_workspace_size(2, 4, 1000, 4, 1)
    assert _call(lib.fvb_beam_search_select, SELECT, dict(ws_bytes=need - 1)) == small
    wide = dict(columns=4096, max_kv=65536, window=65536)  # split over the SMs, so partials are kept
    need = lib.fvb_paged_attention_window_decode_workspace_size(2, 8, 2, 128, 65536, 65536, 4)
    assert need > 0
    assert _call(lib.fvb_paged_attention_window_decode, DECODE, dict(wide, ws_bytes=0)) == small
    assert _call(lib.fvb_paged_attention_window_decode, DECODE, dict(wide, ws=None)) == small


def test_window_workspace_sizes(lib):
    size = lib.fvb_paged_attention_window_decode_workspace_size
    assert size(0, 8, 2, 128, 50, 20, 4) == 0
    assert size(2, 7, 2, 128, 50, 20, 4) == 0 and size(2, 8, 2, 128, 50, 0, 4) == 0
    assert size(4, 8, 2, 64, 4096, 64, 4) == 0  # a few pages: one split, no partials
    assert size(2000, 16, 8, 128, 4096, 64, 4) == 0  # more sequences than the tensor-core kernel's table holds
    # what it takes follows the window, not the context
    assert size(32, 64, 8, 128, 131072, 512, 0) == size(32, 64, 8, 128, 8192, 512, 0)
    # the tensor-core kernel's partials: two cut units a CTA of 16 heads
    assert size(256, 16, 8, 128, 4096, 1024, 4) >= 148 * 2 * 16 * 129 * 4


def test_shared_prefix_workspace_sizes(lib):
    size = lib.fvb_paged_attention_shared_prefix_workspace_size
    assert size(0, 8, 2, 128, 50, 1, 32, 1) == 0
    for dtype in (0, 1, 2):
        assert size(32, 32, 8, 128, 5120, 1, 4096, dtype) >= 32 * 32 * 129 * 4  # a partial of every (sequence, head)
        assert size(100, 8, 2, 64, 64, 3, 48, dtype) == 0  # too small to share anything: one split, no partials


SELECT = dict(logits=16, stride=1000, requests=2, beams=4, vocab=1000, dtype=1, scores=16, finished=None, eos=-1, select=4,
              tokens=16, parents=16, out=16, ws=256, ws_bytes=BIG, stream=None)


@pytest.mark.parametrize("over,status", [
    (dict(dtype=9), UNSUPPORTED),
    (dict(requests=-1), INVALID),
    (dict(beams=0), INVALID),
    (dict(beams=65), UNSUPPORTED),
    (dict(select=0), INVALID),
    (dict(select=65), UNSUPPORTED),
    (dict(vocab=0), INVALID),
    (dict(vocab=1 << 31, stride=1 << 31), UNSUPPORTED),
    (dict(stride=999), INVALID),
    (dict(beams=1, vocab=3, select=4), INVALID),  # fewer candidates than are asked for
    (dict(finished=16, eos=-1), INVALID),
    (dict(finished=16, eos=1000), INVALID),
    (dict(logits=None), INVALID),
    (dict(scores=None), INVALID),
    (dict(out=None), INVALID),
    (dict(logits=17), MISALIGNED),
    (dict(tokens=12), MISALIGNED),
    (dict(scores=18), MISALIGNED),
    (dict(ws=264), MISALIGNED),
    (dict(beams=64, vocab=131072 * 17, stride=131072 * 17), UNSUPPORTED),  # more than 1024 parts a request
])
def test_beam_select_refuses(lib, over, status):
    assert _call(lib.fvb_beam_search_select, SELECT, over) == status


def test_beam_select_workspace_size(lib):
    size = lib.fvb_beam_search_workspace_size
    assert size(0, 4, 1000, 4, 1) == 0 and size(2, 65, 1000, 4, 1) == 0 and size(2, 4, 1000, 4, 9) == 0
    assert size(2, 4, 1000, 4, 1) >= 8 * (4 * 8 + 8)
    assert size(32, 8, 151936, 16, 1) > size(2, 8, 151936, 16, 1)


def _reorder(pools=(16,), **over):
    n = len(pools)
    array = (ctypes.c_void_p * max(n, 1))(*pools)
    base = dict(k=array, v=array, layers=n, num_blocks=10, hkv=2, d=64, page=16, dtype=1, tables=1024, new=4096,
                columns=4, lens=16, parents=16, requests=2, beams=4, stream=None)
    base.update(over)
    return base


@pytest.mark.parametrize("over,status", [
    (dict(dtype=9), UNSUPPORTED),
    (dict(layers=0), INVALID),
    (dict(num_blocks=-1), INVALID),
    (dict(hkv=0), INVALID),
    (dict(page=0), INVALID),
    (dict(beams=0), INVALID),
    (dict(beams=65), UNSUPPORTED),
    (dict(d=4), MISALIGNED),
    (dict(requests=-1), INVALID),
    (dict(k=None), INVALID),
    (dict(lens=None), INVALID),
    (dict(parents=None), INVALID),
    (dict(parents=20), MISALIGNED),
    (dict(tables=None), INVALID),
    (dict(new=1024), INVALID),         # in place
    (dict(new=1024 + 127), INVALID),   # the last byte of 2 * 4 * 4 ids of 4 bytes
    (dict(new=1024 - 127), INVALID),
])
def test_beam_reorder_refuses(lib, over, status):
    assert _call(lib.fvb_beam_reorder_kvcache, _reorder(), over) == status
    assert _call(lib.fvb_beam_reorder_kvcache, _reorder(pools=(16, 24)), {}) == MISALIGNED
    assert _call(lib.fvb_beam_reorder_kvcache, _reorder(pools=(16, None)), {}) == INVALID


def test_operators_are_registered():
    from femtovllm_b200 import _C

    for name in ("PagedAttentionWindowGemvCuda", "PagedAttentionWindowGemmCuda", "PagedAttentionSharedPrefixGemvCuda",
                 "BeamSearchSelectCuda", "BeamReorderKVCacheCuda"):
        assert callable(getattr(_C, name))
    for name in ("paged_attention_window_decode", "paged_attention_window_prefill",
                 "paged_attention_shared_prefix_decode", "beam_search_select", "beam_reorder_kvcache"):
        assert hasattr(torch.ops.femtovllm_b200, name)


def test_operators_refuse_tensors_of_the_cpu():
    i32 = torch.int32
    q, pool = torch.zeros(8, 2, 128), torch.zeros(4, 2, 16, 128)
    tables, lens, cu = torch.zeros(2, 1, dtype=i32), torch.ones(2, dtype=i32), torch.tensor([0, 1, 2], dtype=i32)
    with pytest.raises(ValueError):
        ops.paged_attention_window_gemv(q, pool, pool, tables, lens, 1, 4)
    with pytest.raises(ValueError):
        ops.paged_attention_window_gemm(q, pool, pool, cu, 1, tables, lens, lens - 1, 4)
    with pytest.raises(ValueError):
        ops.paged_attention_shared_prefix_gemv(q, pool, pool, tables, lens, 1, cu, lens, 16)
    with pytest.raises(ValueError):
        ops.beam_search_select(torch.zeros(4, 100), torch.zeros(1, 4), 4)
    with pytest.raises(ValueError):
        ops.beam_reorder_kvcache([pool], [pool], tables, lens, torch.zeros(1, 2, dtype=torch.int64))
