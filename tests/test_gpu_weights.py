"""Softmax weights of the 16-bit window and shared-prefix operators: as good as in 32 bits, large and small.

tests/ref64.py allows each weight the rounding of a single 16-bit operand, u = eps / 2.  Held as two of them, p = hi + lo,
|p - hi| <= u p and lo is rounded once more, so a weight is off by u^2 of itself: ``check`` takes u A out of that bound
and puts u^2 A in (A = sum p |v|, the attention of |v|).  The queries use four dims, which keeps the bound on the scores'
own error (it grows with sum |q k|) far below u, and their scores are spread so that a few keys share the weight.
"""

import numpy as np
import pytest
import torch

import ref64
from femtovllm_b200 import ops, workloads
import test_gpu_shared_prefix as shared
from test_gpu_sharing import wide

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def check(got, q, k, v, *args, **kw):
    out, bound = ref64.attention(q, k, v, *args, **kw)
    a = ref64.attention(q, k, v.abs(), *args, **kw)[0]
    u = torch.finfo(q.dtype).eps / 2
    ref64.check_attention(got, (out, bound - a * (u - u * u)))


def _peaked(q, scale=12.0):
    """Queries of four dims, whose scores have a deviation of 2 * scale / sqrt(d) on unit normal keys."""
    q[..., 4:] = 0
    q.mul_(scale)
    return q


def _pools(blocks, hkv, d, dtype, dev, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn((blocks, hkv, 16, d), generator=gen, device=dev).to(dtype) for _ in range(2)]


def _decode_inputs(lens, hq, hkv, d, dtype, dev, seed):
    pages = (np.asarray(lens) + 15) // 16
    k, v = _pools(int(pages.sum()) + 1, hkv, d, dtype, dev, seed)
    tables = np.full((len(lens), int(pages.max())), -1, np.int32)
    order = np.random.default_rng(seed).permutation(int(pages.sum())).astype(np.int32)
    at = np.concatenate([[0], np.cumsum(pages)])
    for s, n in enumerate(pages):
        tables[s, :n] = order[at[s]: at[s] + n]
    gen = torch.Generator(device=dev).manual_seed(seed + 1)
    q = _peaked(torch.randn((hq, len(lens), d), generator=gen, device=dev).to(dtype))
    return q, k, v, torch.from_numpy(tables).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("n_rep", [1, 2, 4, 5, 8, 12, 16, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_window_decode(dtype, d, n_rep, cuda_device):
    """Batches on either side of the choice between the kernels."""
    for n in (6, 160):
        lens = np.random.default_rng(n).integers(1, 129, size=n)
        lens[:2] = 128, 1
        q, k, v, tables, kv = _decode_inputs(lens, 16 * n_rep, 16, d, dtype, cuda_device, n_rep)
        for window, sinks in ((1 << 30, 0), (100, 3)):
            got = ops.paged_attention_window_gemv(q, k, v, tables, kv, int(lens.max()), window, sinks)
            check(got, q, k, v, tables, kv, window=window, sinks=sinks)


def _one_key_above(k, v, q, page0, log2):
    """Key 0 of `page0` scores `log2` above all others and has a V of zero; the others' V is one."""
    q.zero_()
    k.zero_()
    q[..., 0] = 1.0
    k[page0, :, 0, 0] = log2 * np.log(2.0) * k.shape[3] ** 0.5
    v.fill_(1.0)
    v[page0, :, 0] = 0.0


@pytest.mark.parametrize("log2", [13, 20, 26])
@pytest.mark.parametrize("dtype", DTYPES)
def test_window_decode_of_small_weights_behind_a_sink(dtype, log2, cuda_device):
    """20000 keys whose weights are 2^-log2 of the first one's make up the whole output."""
    for n_rep in (2, 8, 16):
        q, k, v, tables, kv = _decode_inputs([20000], 16 * n_rep, 16, 64, dtype, cuda_device, 3)
        _one_key_above(k, v, q, tables[0, 0].item(), log2)
        got = ops.paged_attention_window_gemv(q, k, v, tables, kv, 20000, 1 << 30, 1)
        check(got, q, k, v, tables, kv, window=1 << 30, sinks=1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_window_decode_with_an_infinite_value(dtype, cuda_device):
    """An infinite V shows as itself in its sequence's column, and nowhere else."""
    q, k, v, tables, kv = _decode_inputs([60] * 800, 32, 16, 64, dtype, cuda_device, 4)
    q.zero_()  # equal weights, none of them rounded
    v.abs_()
    want = ops.paged_attention_window_gemv(q, k, v, tables, kv, 60, 64, 0)
    v[tables[3, 1].item(), 2, 5, 7] = torch.inf
    got = ops.paged_attention_window_gemv(q, k, v, tables, kv, 60, 64, 0)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[4:6, 3, 7] = True
    assert (got[hit] == torch.inf).all() and torch.equal(got[~hit], want[~hit])


def _share(s, **kw):
    _peaked(s["q"])
    for s in (s, wide(s)):
        got = shared.call(s, **kw)
        check(got, s["q"], s["kp"], s["vp"], s["tables"], s["kv"])


GROUPS = [(20, 16), (3, 20)], [30, 77, 150], [60, 1]


@pytest.mark.parametrize("n_rep", [1, 2, 4, 5, 8, 12, 16, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_own_keys_of_sequences_in_groups(dtype, d, n_rep, cuda_device):
    """A bound of 0 on the prefixes leaves every key to its own sequence."""
    _share(shared.make(*GROUPS, 4 * n_rep, 4, d, dtype, cuda_device, seed=n_rep), max_prefix=0)


@pytest.mark.parametrize("log2", [13.3, 20.3, 24.3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_weights_behind_a_sink_in_a_prefill_and_a_prefix(dtype, log2, cuda_device):
    """The same rows on the kernels of 128-row tiles.  A weight of 2^-24.3 still has all of a 16-bit operand's bits."""
    for n_rep in (2, 8):
        b = workloads.custom([6000, 900], [200, 33], 4 * n_rep, 4, 64, dtype, seed=2).materialize(cuda_device)
        md = b.device_metadata(cuda_device)
        k, v, tables = b.k_pool, b.v_pool, md["block_tables"]
        _one_key_above(k, v, b.q, tables[0, 0].item(), log2)
        got = ops.paged_attention_window_gemm(b.q, k, v, md["cu_seqlens"], 200, tables, md["kv_lens"], md["positions"],
                                              1 << 30, 1)
        ref64.check_attention(got, ref64.attention(b.q, k, v, tables, md["kv_lens"], md["cu_seqlens"], md["positions"],
                                                   1 << 30, 1))
        s = wide(shared.make([(3, 8000)], [5, 300, 20], [], 4 * n_rep, 4, 64, dtype, cuda_device, seed=2))
        _one_key_above(s["kp"], s["vp"], s["q"], s["tables"][0, 0].item(), log2)
        ref64.check_attention(shared.call(s), ref64.attention(s["q"], s["kp"], s["vp"], s["tables"], s["kv"]))


@pytest.mark.parametrize("n_rep", [1, 2, 4, 5, 8, 12, 16, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_prefixes(dtype, d, n_rep, cuda_device):
    """Groups of one query tile and of several, prefixes of a page, of part of a tile and of several splits."""
    for i, shape in enumerate([GROUPS, ([(5, 120), (9, 700), (2, 64)], [1, 20], [33]), ([(3, 2000)], [4], []),
                               ([(150, 100)], [2], [])]):
        _share(shared.make(*shape, 4 * n_rep, 4, d, dtype, cuda_device, seed=n_rep + i))
