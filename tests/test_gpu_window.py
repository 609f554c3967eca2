"""Window-with-sinks attention on the GPU against the plain form in 64 bits (tests/ref64.py).

Pages that no query sees are -1 in the tables or full of NaN in the pool, and so are the keys between sinks and
window inside pages that are read; every comparison therefore also shows that nothing of them leaks in.
"""

import math

import numpy as np
import pytest
import torch

import ref64
from femtovllm_b200 import ops, workloads

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 257, 1000, 2049, 5000]
MASKS = [(1, 0), (1, 5), (16, 0), (17, 1), (100, 20), (128, 16), (700, 129), (2048, 4), (1 << 30, 0), (64, 1 << 30)]
GQA = [1, 2, 3, 4, 5, 8, 16]


def _poisoned(b, first, window, sinks, drop):
    """Pools with NaN in every key no query of its sequence sees; tables with -1 for wholly unseen pages."""
    kp, vp = b.k_pool.clone(), b.v_pool.clone()
    tables = torch.from_numpy(b.block_tables).to(kp.device)
    for s, n in enumerate(b.kv_lens.tolist()):
        key = torch.arange(((n + 15) // 16) * 16, device=kp.device)
        lo = max(0, first[s] - window + 1)
        seen = ((key >= lo) | (key < sinks)) & (key < n)
        pages = tables[s, : len(key) // 16].long()
        for pool in (kp, vp):
            rows = pool[pages]
            rows.masked_fill_(~seen.view(-1, 1, 16, 1), math.nan)
            pool[pages] = rows
        if drop:
            unseen = ~seen.view(-1, 16).any(1)
            tables[s, : len(unseen)][unseen] = -1
    return kp, vp, tables


def _decode(b, window, sinks, drop=True, **kw):
    kp, vp, tables = _poisoned(b, (b.kv_lens - 1).tolist(), window, sinks, drop)
    lens = torch.from_numpy(b.kv_lens).to(kp.device)
    got = ops.paged_attention_window_gemv(b.q, kp, vp, tables, lens, b.max_kv_len, window, sinks, **kw)
    ref64.check_attention(got, ref64.attention(b.q, kp, vp, tables, lens, window=window, sinks=sinks),
                          f"window {window} sinks {sinks}")
    assert ops.read_device_error() == (0, 0)
    return got


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_sweep(dtype, head_dim, n_rep, cuda_device):
    lens = np.random.default_rng(n_rep).permutation(LENS)
    b = workloads.custom(lens, np.ones(len(lens)), 2 * n_rep, 2, head_dim, dtype, seed=n_rep).materialize(cuda_device)
    for i, (window, sinks) in enumerate(MASKS):
        _decode(b, window, sinks, drop=i % 2 == 0)


@pytest.mark.parametrize("n_rep", [2, 8])
def test_decode_many_short_sequences_without_splits(n_rep, cuda_device):
    lens = np.random.default_rng(0).integers(1, 700, size=300)
    b = workloads.custom(lens, np.ones(300), 8 * n_rep, 8, 128, torch.bfloat16, seed=3).materialize(cuda_device)
    _decode(b, 128, 4)


@pytest.mark.parametrize("dtype,n_rep", [(torch.bfloat16, 4), (torch.float16, 8), (torch.float32, 8)])
def test_decode_long_context_splits(dtype, n_rep, cuda_device):
    b = workloads.custom([70000, 33333], [1, 1], 2 * n_rep, 2, 128, dtype, seed=4).materialize(cuda_device)
    for window, sinks in [(4096, 128), (30001, 3), (1 << 30, 7)]:
        _decode(b, window, sinks)


def test_decode_views_and_layouts(cuda_device):
    b = workloads.custom([40, 300, 77], [1, 1, 1], 16, 8, 128, torch.bfloat16, seed=5).materialize(cuda_device)
    plain = _decode(b, 50, 3)
    wide = torch.zeros(3, 40 * 128, dtype=torch.bfloat16, device=cuda_device)  # q inside a wider projection
    wide[:, : 16 * 128] = b.q.transpose(0, 1).reshape(3, -1)
    b.q = wide[:, : 16 * 128].view(3, 16, 128).transpose(0, 1)
    got = _decode(b, 50, 3, out_token_major=True)
    assert torch.equal(got, plain) and got.transpose(0, 1).is_contiguous()


def test_decode_empty_context_and_no_sequences(cuda_device):
    b = workloads.custom([5, 20], [1, 1], 8, 2, 64, torch.bfloat16, seed=6).materialize(cuda_device)
    tables = torch.from_numpy(b.block_tables).to(cuda_device)
    lens = torch.tensor([0, 20], dtype=torch.int32, device=cuda_device)
    got = ops.paged_attention_window_gemv(b.q, b.k_pool, b.v_pool, tables, lens, 20, 4, 2)
    assert (got[:, 0] == 0).all()
    ref64.check_attention(got, ref64.attention(b.q, b.k_pool, b.v_pool, tables, lens, window=4, sinks=2))
    none = ops.paged_attention_window_gemv(b.q[:, :0], b.k_pool, b.v_pool, tables[:0], lens[:0], 0, 4, 2)
    assert none.shape == (8, 0, 64)


def test_decode_in_a_pool_past_32_bit_offsets(cuda_device):
    num_blocks, hkv, d = 135000, 8, 128  # 2.2e9 elements a pool
    kp = torch.empty(num_blocks, hkv, 16, d, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.empty_like(kp)
    pages = torch.arange(num_blocks - 40, num_blocks, device=cuda_device)
    kp[pages] = torch.randn(40, hkv, 16, d, device=cuda_device).to(torch.bfloat16)
    vp[pages] = torch.randn(40, hkv, 16, d, device=cuda_device).to(torch.bfloat16)
    tables = pages.view(2, 20).int().contiguous()
    lens = torch.tensor([320, 301], dtype=torch.int32, device=cuda_device)
    for heads in (16, 64):
        q = torch.randn(heads, 2, d, device=cuda_device).to(torch.bfloat16)
        got = ops.paged_attention_window_gemv(q, kp, vp, tables, lens, 320, 100, 20)
        ref64.check_attention(got, ref64.attention(q, kp, vp, tables, lens, window=100, sinks=20))


def test_decode_bad_page_inside_the_window_is_reported(cuda_device):
    b = workloads.custom([100], [1], 16, 8, 128, torch.bfloat16, seed=8).materialize(cuda_device)
    tables = torch.from_numpy(b.block_tables).to(cuda_device)
    lens = torch.from_numpy(b.kv_lens).to(cuda_device)
    for column, code in [(6, 7), (2, 0)]:  # pages 5 and 6 hold the last 20 keys; page 2 holds none
        bad = tables.clone()
        bad[0, column] = -1
        ops.paged_attention_window_gemv(b.q, b.k_pool, b.v_pool, bad, lens, 100, 20, 0)
        assert ops.read_device_error()[0] == code


# ------------------------------------------------------------------ prefill


def _prefill(b, window, sinks, drop=True):
    first = (b.kv_lens - b.q_lens).tolist()
    kp, vp, tables = _poisoned(b, first, window, sinks, drop)
    md = b.device_metadata(kp.device)
    got = ops.paged_attention_window_gemm(b.q, kp, vp, md["cu_seqlens"], b.max_q_len, tables, md["kv_lens"],
                                          md["positions"], window, sinks)
    want = ref64.attention(b.q, kp, vp, tables, md["kv_lens"], md["cu_seqlens"], md["positions"], window, sinks)
    ref64.check_attention(got, want, f"window {window} sinks {sinks}")
    assert ops.read_device_error() == (0, 0)


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_sweep(dtype, head_dim, n_rep, cuda_device):
    q_lens = np.array([1, 130, 1, 33, 300, 2, 64, 1, 257])
    kv = q_lens + np.array([0, 0, 500, 17, 900, 2000, 64, 1, 15])
    b = workloads.custom(kv, q_lens, 2 * n_rep, 2, head_dim, dtype, seed=n_rep).materialize(cuda_device)
    for i, (window, sinks) in enumerate(MASKS):
        _prefill(b, window, sinks, drop=i % 2 == 1)


def test_prefill_long_chunk_over_a_prefix(cuda_device):
    b = workloads.custom([5000, 3000], [1500, 800], 16, 8, 128, torch.bfloat16, seed=9).materialize(cuda_device)
    for window, sinks in [(1000, 4), (129, 300), (4000, 0)]:
        _prefill(b, window, sinks)


@pytest.mark.parametrize("dtype,n_rep", [(torch.float32, 2), (torch.bfloat16, 2), (torch.bfloat16, 8)])
def test_prefill_rows_whose_mask_leaves_nothing_are_zero(dtype, n_rep, cuda_device):
    # kv_len below the positions: the later queries' windows lie wholly behind the last key.
    b = workloads.custom([100, 40, 60], [60, 40, 1], 2 * n_rep, 2, 64, dtype, seed=10).materialize(cuda_device)
    md = b.device_metadata(cuda_device)
    kv = torch.tensor([70, 40, 30], dtype=torch.int32, device=cuda_device)
    for sinks in (0, 3):
        got = ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 60, md["block_tables"], kv,
                                              md["positions"], 10, sinks)
        want = ref64.attention(b.q, b.k_pool, b.v_pool, md["block_tables"], kv, md["cu_seqlens"], md["positions"],
                               10, sinks)
        assert sinks > 0 or (want[0][:, 45:60] == 0).all()
        ref64.check_attention(got, want, f"sinks {sinks}")
    assert ops.read_device_error() == (0, 0)


def test_prefill_equals_decode_for_single_tokens(cuda_device):
    for n_rep in (2, 8):
        b = workloads.custom([300, 17, 900], [1, 1, 1], 8 * n_rep, 8, 128, torch.bfloat16, seed=11).materialize(cuda_device)
        md = b.device_metadata(cuda_device)
        a = ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 1, md["block_tables"],
                                            md["kv_lens"], md["positions"], 128, 4)
        ref64.check_attention(a, ref64.attention(b.q, b.k_pool, b.v_pool, md["block_tables"], md["kv_lens"],
                                                 window=128, sinks=4))


# ------------------------------------------------------------------ graphs, streams, a running window


def test_window_ops_replay_in_a_graph_and_run_on_two_streams(cuda_device):
    q_lens = np.array([1, 64, 1, 200, 33])
    b = workloads.custom(q_lens + 700, q_lens, 16, 8, 128, torch.bfloat16, seed=12).materialize(cuda_device)
    md = b.device_metadata(cuda_device)
    q1 = b.q[:, :5].contiguous()

    def both():
        return (ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 200, md["block_tables"],
                                                md["kv_lens"], md["positions"], 128, 4),
                ops.paged_attention_window_gemv(q1, b.k_pool, b.v_pool, md["block_tables"], md["kv_lens"],
                                                b.max_kv_len, 300, 4))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = both()
    for it in range(3):
        b.q.copy_(torch.randn_like(b.q, dtype=torch.float32).to(b.q.dtype))
        q1.copy_(b.q[:, 7:12])
        torch.cuda.synchronize()
        want = both()
        g.replay()
        with torch.cuda.stream(side):  # an eager call beside the replay
            side.wait_stream(torch.cuda.current_stream())
            again = both()
        torch.cuda.synchronize()
        for a, w, e in zip(got, want, again):
            assert torch.equal(a, w) and torch.equal(e, w)
    del g


def test_running_window_with_pages_taken_back(cuda_device):
    """Sequences grow token by token in a small pool: pages behind the window go back and are handed out again."""
    window, sinks, hq, hkv, d, steps = 40, 5, 8, 4, 64, 200
    gen = torch.Generator(device=cuda_device).manual_seed(0)
    num_blocks = 2 * (1 + 4)  # per sequence: one sink page, four window pages
    kp = torch.full((num_blocks, hkv, 16, d), math.nan, device=cuda_device, dtype=torch.bfloat16)
    vp = kp.clone()
    free = list(range(num_blocks))
    tables = torch.full((2, 16), -1, dtype=torch.int32)
    ks, vs = [], []
    for n in range(steps):
        k = torch.randn(2, hkv, d, generator=gen, device=cuda_device).to(torch.bfloat16)
        v = torch.randn(2, hkv, d, generator=gen, device=cuda_device).to(torch.bfloat16)
        ks.append(k), vs.append(v)
        if n % 16 == 0:
            for s in range(2):
                gone = (n - window + 1) // 16 - 1  # last page whose keys lie behind the window from here on
                if gone >= 1 and tables[s, gone] >= 0:
                    free.append(int(tables[s, gone]))
                    tables[s, gone] = -1
                tables[s, n // 16] = free.pop(0)
        tab = tables.to(cuda_device)
        at = torch.full((2,), n, dtype=torch.int32, device=cuda_device)
        ops.store_kvcache(k, v, kp, vp, ops.build_slot_mapping(at, tab))
        q = torch.randn(hq, 2, d, generator=gen, device=cuda_device).to(torch.bfloat16)
        got = ops.paged_attention_window_gemv(q, kp, vp, tab, at + 1, 256, window, sinks)
        if n % 7 and n < steps - 3:
            continue
        seen = [j for j in range(n + 1) if n - j < window or j < sinks]
        kd = torch.stack([ks[j] for j in seen], 2).double()  # (2, hkv, n, d)
        vd = torch.stack([vs[j] for j in seen], 2).double()
        x = torch.einsum("hgbd,bhnd->bhgn", q.double().view(hkv, 2, 2, d), kd) / math.sqrt(d)
        p = torch.softmax(x, -1)
        want = torch.einsum("bhgn,bhnd->hgbd", p, vd).reshape(hq, 2, d)
        size = torch.einsum("bhgn,bhnd->hgbd", p, vd.abs()).reshape(hq, 2, d)
        # Each weight is rounded to bf16 before P V, off by at most 2^-8 of itself, so the sum by at most
        # 2^-8 sum p |v|; the output is rounded again; scores in 32 bits are far below that.
        assert ((got.double() - want).abs() <= size * 2.0**-8 + want.abs() * 2.0**-8 + 1e-4).all(), n
    assert ops.read_device_error() == (0, 0)
