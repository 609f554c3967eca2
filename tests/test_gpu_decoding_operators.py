"""The window, shared-prefix and beam operators where another kernel, tile or path takes over, against the plain forms
in 64 bits."""

import ctypes
import math

import numpy as np
import pytest
import torch

import cabi
import ref64
from femtovllm_b200 import capi, ops, workloads
import test_gpu_shared_prefix as shared
from test_gpu_beam import check as check_select
from test_gpu_window import GQA, _decode, _prefill

pytestmark = pytest.mark.gpu


def _workspace(b, window, sinks):
    return cabi.lib().fvb_paged_attention_window_decode_workspace_size(
        len(b.kv_lens), b.q.shape[0], b.k_pool.shape[1], b.q.shape[2], b.max_kv_len, window, sinks)


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
def test_window_decode_of_a_crowd(head_dim, n_rep, cuda_device):
    """Enough pages an SM for the tensor-core kernel, units of one tile to three, cut wherever the SMs' shares end."""
    dtype = torch.float16 if n_rep % 2 else torch.bfloat16
    lens = np.random.default_rng(n_rep).integers(1, 260, size=1024)
    lens[:20] = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 130, 255, 256, 257, 1, 1, 1, 259, 259]
    b = workloads.custom(lens, np.ones(1024), 8 * n_rep, 8, head_dim, dtype, seed=n_rep).materialize(cuda_device)
    for i, (window, sinks) in enumerate([(33, 1), (17, 20), (1 << 30, 0)]):
        assert _workspace(b, window, sinks) > 0  # (the split-KV kernel would take one split and keep no partials)
        _decode(b, window, sinks, drop=i % 2 == 0)


@pytest.mark.parametrize("n_rep", [1, 8])
def test_window_decode_at_the_border_between_the_kernels(n_rep, cuda_device):
    """The same sequences in batches on either side of the rule, and of the largest table."""
    for n in (290, 1024, 1025, 1100):
        lens = np.random.default_rng(n).integers(1, 90, size=n)
        b = workloads.custom(lens, np.ones(n), 8 * n_rep, 8, 64, torch.bfloat16, seed=n).materialize(cuda_device)
        _decode(b, 20, 3)


def test_window_decode_with_empty_sequences_in_a_crowd(cuda_device):
    lens = np.random.default_rng(5).integers(1, 400, size=600)
    b = workloads.custom(lens, np.ones(600), 16, 8, 128, torch.bfloat16, seed=5).materialize(cuda_device)
    tables = torch.from_numpy(b.block_tables).to(cuda_device)
    kv = torch.from_numpy(b.kv_lens).to(cuda_device)
    kv[::7] = 0
    got = ops.paged_attention_window_gemv(b.q, b.k_pool, b.v_pool, tables, kv, 400, 300, 2)
    ref64.check_attention(got, ref64.attention(b.q, b.k_pool, b.v_pool, tables, kv, window=300, sinks=2))
    assert (got[:, ::7] == 0).all()


def _special_keys(k_pool, table, keys, value):
    """A copy of the pool with `value` in all of a sequence's `keys`."""
    k = k_pool.clone()
    keys = torch.as_tensor(keys, device=k.device)
    k[table[keys // 16].long(), :, keys % 16] = value
    return k


@pytest.mark.parametrize("dtype,n_rep,n", [(torch.bfloat16, 2, 700), (torch.bfloat16, 8, 700), (torch.bfloat16, 2, 5),
                                           (torch.bfloat16, 8, 5), (torch.float32, 2, 5), (torch.float32, 2, 300)])
def test_window_decode_with_infinite_and_nan_keys(dtype, n_rep, n, cuda_device):
    """Scores of -inf weigh nothing wherever they stand, also where they fill a tile; a NaN shows in its sequence only."""
    lens = np.full(n, 400)
    b = workloads.custom(lens, np.ones(n), 8 * n_rep, 8, 64, dtype, seed=8).materialize(cuda_device)
    b.q.abs_().clamp_(min=0.01)
    tables, kv = torch.from_numpy(b.block_tables).to(cuda_device), torch.from_numpy(b.kv_lens).to(cuda_device)
    run = lambda k: ops.paged_attention_window_gemv(b.q, k, b.v_pool, tables, kv, 400, 390, 3)  # noqa: E731
    k = b.k_pool
    for s, keys in [(0, range(0, 130)), (1, range(120, 300)), (2, range(256, 400)), (3, [399])]:
        k = _special_keys(k, tables[s], list(keys), -math.inf)
    low = torch.where(k == -math.inf, torch.full_like(k, -1e4), k)  # far below the others' scores: the same weights
    got, same = run(k), run(low)
    assert torch.isfinite(got).all()
    ref64.check_attention(got, ref64.attention(b.q, low, b.v_pool, tables, kv, window=390, sinks=3))
    ref64.check_attention(same, ref64.attention(b.q, low, b.v_pool, tables, kv, window=390, sinks=3))
    bad = torch.isnan(run(_special_keys(b.k_pool, tables[4], [200], math.nan)))
    assert bad[:, 4].all() and not bad[:, :4].any() and not bad[:, 5:].any()


@pytest.mark.parametrize("dtype,n_rep", [(torch.float32, 2), (torch.bfloat16, 2), (torch.bfloat16, 8)])
def test_window_prefill_with_infinite_and_nan_keys(dtype, n_rep, cuda_device):
    b = workloads.custom([400, 300], [200, 30], 4 * n_rep, 4, 64, dtype, seed=8).materialize(cuda_device)
    md = b.device_metadata(cuda_device)
    b.q.abs_().clamp_(min=0.01)
    tables = md["block_tables"]

    def run(k):
        return ops.paged_attention_window_gemm(b.q, k, b.v_pool, md["cu_seqlens"], 200, tables, md["kv_lens"],
                                               md["positions"], 150, 3)

    k = _special_keys(b.k_pool, tables[0], list(range(40, 199)) + [0, 1, 2], -math.inf)
    low = torch.where(k == -math.inf, torch.full_like(k, -1e4), k)
    got = run(k)
    ref64.check_attention(got, ref64.attention(b.q, low, b.v_pool, tables, md["kv_lens"], md["cu_seqlens"],
                                               md["positions"], 150, 3))
    bad = torch.isnan(run(_special_keys(b.k_pool, tables[0], [210], math.nan)))
    sees = (md["positions"][:200] >= 210) & (md["positions"][:200] < 210 + 150)
    assert bad[:, :200][:, sees].all() and not bad[:, :200][:, ~sees].any() and not bad[:, 200:].any()


# ------------------------------------------------------------------ fp32 prefill


@pytest.mark.parametrize("n_rep", [1, 3, 8, 16])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_fp32_prefill_keys_shared_by_a_cluster(head_dim, n_rep, cuda_device):
    b = workloads.custom([9000, 700, 5003], [40, 1, 16], n_rep, 1, head_dim, torch.float32, seed=1).materialize(cuda_device)
    for window, sinks in [(1 << 30, 0), (4096, 130), (33, 7000), (600, 0), (1, 0)]:
        _prefill(b, window, sinks)


@pytest.mark.parametrize("n_rep", [1, 5])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_fp32_prefill_large_tiles(head_dim, n_rep, cuda_device):
    q_lens = np.array([900, 1, 64, 63, 65, 450, 16, 17, 2])
    kv = q_lens + np.array([300, 800, 0, 64, 1, 0, 15, 100, 31])
    b = workloads.custom(kv, q_lens, 8 * n_rep, 8, head_dim, torch.float32, seed=2).materialize(cuda_device)
    for window, sinks in [(200, 4), (1000, 0), (15, 70)]:
        _prefill(b, window, sinks, drop=False)


def test_fp32_prefill_scores_far_apart_and_infinite(cuda_device):
    """Rows whose running maximum moves by thousands, keys whose score is -inf, and one whose score is +inf (NaN out)."""
    b = workloads.custom([300, 90], [200, 1], 4, 2, 64, torch.float32, seed=3).materialize(cuda_device)
    b.q.mul_(40)
    _prefill(b, 128, 4)
    md = b.device_metadata(cuda_device)
    k = b.k_pool.clone()
    page = int(b.block_tables[0, 3])
    k[page, :, 5] = -math.inf  # key 53 of the first sequence: scores of -inf, +inf or NaN, by the query
    q = b.q.abs()              # here -inf for every query
    got = ops.paged_attention_window_gemm(q, k, b.v_pool, md["cu_seqlens"], 200, md["block_tables"], md["kv_lens"],
                                          md["positions"], 128, 0)
    small = k.clone()
    small[page, :, 5] = -3e30  # below every other score by far: the same weights
    same = ops.paged_attention_window_gemm(q, small, b.v_pool, md["cu_seqlens"], 200, md["block_tables"],
                                           md["kv_lens"], md["positions"], 128, 0)
    assert torch.equal(got, same) and torch.isfinite(got).all()
    k[page, :, 5] = math.inf
    got = ops.paged_attention_window_gemm(q, k, b.v_pool, md["cu_seqlens"], 200, md["block_tables"], md["kv_lens"],
                                          md["positions"], 128, 0)
    sees = (md["positions"][:200] >= 53) & (md["positions"][:200] < 53 + 128)
    assert torch.isnan(got[:, :200][:, sees]).all() and torch.isfinite(got[:, :200][:, ~sees]).all()
    assert torch.isfinite(got[:, 200:]).all()


@pytest.mark.parametrize("dtype,n_rep", [(torch.float32, 2), (torch.bfloat16, 2), (torch.bfloat16, 8)])
def test_window_prefill_leaves_rows_behind_the_last_sequence(dtype, n_rep, cuda_device):
    b = workloads.custom([100, 30, 40], [60, 1, 7], 2 * n_rep, 2, 64, dtype, seed=4).materialize(cuda_device)
    md = b.device_metadata(cuda_device)
    hq, t, d = b.q.shape
    q = torch.cat([b.q, b.q[:, :5]], 1).contiguous()
    out = torch.full_like(q, 7.0)
    lib = cabi.lib()
    need = lib.fvb_paged_attention_prefill_workspace_size(3, hq, 2, d, t + 5, 60)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=cuda_device)
    capi.check(lib.fvb_paged_attention_window_prefill(
        q.data_ptr(), d, (t + 5) * d, out.data_ptr(), d, (t + 5) * d, b.k_pool.data_ptr(), b.v_pool.data_ptr(),
        b.k_pool.shape[0], hq, 2, d, 16, 3, t + 5, md["cu_seqlens"].data_ptr(), 60, md["block_tables"].data_ptr(),
        md["block_tables"].shape[1], md["kv_lens"].data_ptr(), md["positions"].data_ptr(), 50, 3,
        capi.dtype_code(dtype), ws.data_ptr(), need, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "window")
    ref64.check_attention(out[:, :t], ref64.attention(b.q, b.k_pool, b.v_pool, md["block_tables"], md["kv_lens"],
                                                      md["cu_seqlens"], md["positions"], 50, 3))
    assert (out[:, t:] == 7.0).all()


@pytest.mark.parametrize("n_rep", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("window", [60, 100])
def test_window_prefill_single_rows_are_written_once(window, n_rep, cuda_device):
    """Single-token rows of a mixed batch: bit for bit what they are in a batch of their own, whatever runs beside them."""
    q_lens = np.array([1, 400, 1, 1, 700, 33, 1, 2, 1, 900])
    kv = q_lens + np.array([700, 300, 5, 0, 900, 64, 100, 9, 333, 0])
    b = workloads.custom(kv, q_lens, 4 * n_rep, 4, 128, torch.bfloat16, seed=9).materialize(cuda_device)
    md = b.device_metadata(cuda_device)
    ones = np.flatnonzero(q_lens == 1)
    rows = torch.from_numpy(np.concatenate([[0], np.cumsum(q_lens)])[ones]).to(cuda_device)
    pick = torch.from_numpy(ones).to(cuda_device)
    alone = ops.paged_attention_window_gemm(
        b.q[:, rows].contiguous(), b.k_pool, b.v_pool, torch.arange(len(ones) + 1, dtype=torch.int32, device=cuda_device),
        1, md["block_tables"][pick].contiguous(), md["kv_lens"][pick].contiguous(),
        md["positions"][rows].contiguous(), window, 3)
    want = ref64.attention(b.q, b.k_pool, b.v_pool, md["block_tables"], md["kv_lens"], md["cu_seqlens"],
                           md["positions"], window, 3)
    for _ in range(20):
        got = ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 900, md["block_tables"],
                                              md["kv_lens"], md["positions"], window, 3)
        assert torch.equal(got[:, rows], alone)
    ref64.check_attention(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_window_prefill_reports_bad_pages_and_long_contexts(dtype, cuda_device):
    b = workloads.custom([100, 50], [20, 50], 4, 2, 64, dtype, seed=6).materialize(cuda_device)
    md = b.device_metadata(cuda_device)

    def run(tables, lens):
        ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 50, tables, lens, md["positions"],
                                        30, 0)
        return ops.read_device_error()

    assert run(md["block_tables"], md["kv_lens"]) == (0, 0)
    for bad in (-1, -2, b.k_pool.shape[0], 1 << 30):
        tables = md["block_tables"].clone()
        tables[0, 5] = bad
        assert run(tables, md["kv_lens"]) == (7, 0)
        tables = md["block_tables"].clone()
        tables[0, 1] = bad  # keys 16 to 31: behind every query's window
        assert run(tables, md["kv_lens"]) == (0, 0)
    longer = md["kv_lens"].clone()
    longer[1] = 16 * md["block_tables"].shape[1] + 1
    assert run(md["block_tables"], longer) == (1, 1)


def test_fp32_window_prefill_in_two_graphs_and_beside_them(cuda_device):
    b = workloads.custom([900, 300], [100, 40], 8, 2, 128, torch.float32, seed=7).materialize(cuda_device)
    md = b.device_metadata(cuda_device)

    def run(window):
        return ops.paged_attention_window_gemm(b.q, b.k_pool, b.v_pool, md["cu_seqlens"], 100, md["block_tables"],
                                               md["kv_lens"], md["positions"], window, 2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(64)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for window in (64, 700):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(window)
        graphs.append((g, out, window))
    for _ in range(2):
        b.q.normal_()
        torch.cuda.synchronize()
        for g, _, _ in graphs:
            g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            beside = run(700)
        torch.cuda.synchronize()
        for _, out, window in graphs:
            assert torch.equal(out, run(window))
        assert torch.equal(beside, run(700))
    graphs.clear()


# ------------------------------------------------------------------ shared prefixes


def _wide(s, columns=8192):
    """The same call with a table and a bound on kv_lens so wide that it is worth sharing."""
    tables = torch.full((len(s["tables"]), columns), -1, dtype=torch.int32, device=s["tables"].device)
    tables[:, : s["tables"].shape[1]] = s["tables"]
    dtype = capi.dtype_code(s["q"].dtype)
    hq, b, d = s["q"].shape
    args = (b, hq, s["kp"].shape[1], d)
    size = cabi.lib().fvb_paged_attention_shared_prefix_workspace_size
    s = dict(s, tables=tables, max_kv=16 * columns)
    # partials of the shared keys for every (sequence, head): more than each one's own splits would take
    assert size(*args, s["max_kv"], len(s["prefix"]), s["max_prefix"], dtype) > 0
    return s


@pytest.mark.parametrize("n_rep", [1, 2, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_shared_prefix_sweep_with_sharing(dtype, head_dim, n_rep, cuda_device):
    for i, (groups, own, loners) in enumerate(shared.SHAPES):
        shared.check(_wide(shared.make(groups, own, loners, 2 * n_rep, 2, head_dim, dtype, cuda_device, seed=i)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_shared_prefix_of_short_empty_and_skewed_sequences_with_sharing(dtype, cuda_device):
    for seed, shorter in enumerate([{1: 5}, {0: 20, 2: 300}, {0: 0, 3: 0}, {3: 1}, {0: 0, 1: 0, 2: 0, 3: 0}]):
        s = shared.make([(4, 500)], [1, 30], [], 8, 2, 128, dtype, cuda_device, seed=seed, shorter=shorter)
        got = shared.check(_wide(s))
        for b, n in shorter.items():
            assert n > 0 or (got[:, b] == 0).all()
    shared.check(_wide(shared.make([(20, 320)], [1], [20000], 16, 8, 128, dtype, cuda_device, seed=7)))
    s = shared.make([(6, 400), (3, 90)], [5, 50], [7], 8, 4, 64, dtype, cuda_device, seed=3)
    for bound in (0, 10, 100, 399):
        shared.check(_wide(s), max_prefix=bound)


def test_shared_prefix_of_many_sequences_and_groups_with_sharing(cuda_device):
    bf16 = torch.bfloat16
    shared.check(_wide(shared.make([(700, 40), (801, 33)], [1, 20, 3], [9] * 30, 4, 2, 64, bf16, cuda_device, seed=5), 512))
    many = [(2 + i % 3, 16 * (1 + i % 5) + i % 7) for i in range(70)]
    shared.check(_wide(shared.make(many, [1, 20, 3], [], 8, 4, 64, bf16, cuda_device, seed=6), 2048))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_prefix_with_sharing_reports_malformed_groups(dtype, cuda_device):
    s = _wide(shared.make([(4, 100), (4, 100)], [9], [], 16, 8, 128, dtype, cuda_device, seed=9))
    for cu in ([0, 9, 8], [-3, 4, 8], [0, 4, 100], [5, 2, 8]):
        shared.call(dict(s, cu=torch.tensor(cu, dtype=torch.int32, device=cuda_device)))
        assert ops.read_device_error()[0] == 1
    shared.call(dict(s, prefix=torch.tensor([-1, 100], dtype=torch.int32, device=cuda_device)))
    assert ops.read_device_error()[0] == 1
    for bad in (1 << 28, -1, -2):
        tables = s["tables"].clone()
        tables[0, 2] = bad  # the group's first row names its shared pages
        shared.call(dict(s, tables=tables))
        assert ops.read_device_error()[0] == 7
        tables = s["tables"].clone()
        tables[1, 2] = bad  # another row's entry for a shared page is not read
        shared.call(dict(s, tables=tables))
        assert ops.read_device_error()[0] == 0


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_prefix_with_infinite_and_nan_keys(dtype, wide, cuda_device):
    s = shared.make([(6, 640)], [300], [200], 16, 8, 64, dtype, cuda_device, seed=11)
    s = _wide(s) if wide else s
    s["q"].abs_().clamp_(min=0.01)
    k = _special_keys(s["kp"], s["tables"][0], list(range(100, 640)), -math.inf)  # shared: whole tiles and splits
    k = _special_keys(k, s["tables"][1], list(range(640, 800)), -math.inf)
    k = _special_keys(k, s["tables"][2], list(range(640, 940)), -math.inf)
    low = torch.where(k == -math.inf, torch.full_like(k, -1e4), k)
    got = shared.call(dict(s, kp=k))
    ref64.check_attention(got, ref64.attention(s["q"], low, s["vp"], s["tables"], s["kv"]))
    bad = torch.isnan(shared.call(dict(s, kp=_special_keys(s["kp"], s["tables"][3], [700], math.nan))))
    assert bad[:, 3].all() and not bad[:, :3].any() and not bad[:, 4:].any()
    bad = torch.isnan(shared.call(dict(s, kp=_special_keys(s["kp"], s["tables"][3], [17], math.nan))))
    assert bad[:, :6].all() and not bad[:, 6:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_prefix_with_sharing_replays_in_a_graph_and_beside_it(dtype, cuda_device):
    s = _wide(shared.make([(12, 900), (3, 64)], [9, 100, 31], [40], 16, 8, 128, dtype, cuda_device, seed=10))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        shared.call(s)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = shared.call(s)
    for _ in range(3):
        s["q"].normal_()
        torch.cuda.synchronize()
        want = shared.call(s)
        g.replay()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            beside = shared.call(s)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(beside, want)
    del g


# ------------------------------------------------------------------ beam selection


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_with_the_largest_logits_in_few_threads(dtype, cuda_device):
    """Rows of one part each whose thousands of largest logits lie with a few lanes: the bound misses them."""
    n, w, v = 150, 4, 100000
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    logits = torch.randn(n * w, v, generator=gen, device=cuda_device)
    per = 128 // torch.finfo(dtype).bits  # logits of a vector
    high = (torch.arange(v, device=cuda_device) // per) % 128 < 7
    logits[:, high] += 12
    scores = -torch.rand(n, w, generator=gen, device=cuda_device)
    check_select(logits.to(dtype), scores, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [1420, 8200, 16500, 17823, 50001])
def test_select_with_short_last_parts(dtype, v, cuda_device):
    """Vocabularies whose parts end in a few vectors, at every alignment of the rows and for many and few of them."""
    gen = torch.Generator(device=cuda_device).manual_seed(v)
    for n, w, k in [(1, 10, 10), (3, 16, 32), (25, 10, 20), (1, 1, 64), (60, 10, 33)]:
        logits = (torch.randn(n * w, v, generator=gen, device=cuda_device) * 2.5).to(dtype)
        logits[:, v - 40:] += 3  # the short part holds some of the best
        check_select(logits, -torch.rand(n, w, generator=gen, device=cuda_device) * 5, k)
