"""Shared-prefix decode attention on the GPU against the plain form in 64 bits (tests/ref64.py)."""

import math

import numpy as np
import pytest
import torch

import ref64
from femtovllm_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(groups, own, loners, hq, hkv, d, dtype, dev, seed=0, shorter=()):
    """groups: list of (sequences, prefix keys); own / loners: keys behind the prefix / of sequences alone.

    `shorter`: {sequence: kv_len} below its prefix.  Slots past every kv_len hold NaN.
    """
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum([n for n, _ in groups])]).astype(np.int32)
    prefix = np.array([p for _, p in groups], np.int32)
    b = int(cu[-1]) + len(loners)
    kv = np.zeros(b, np.int64)
    for g in range(len(groups)):
        kv[cu[g]:cu[g + 1]] = prefix[g]
    kv[: cu[-1]] += np.resize(np.asarray(own), cu[-1]) if cu[-1] else 0
    kv[cu[-1]:] = loners
    for s, n in dict(shorter).items():
        kv[s] = n
    need = np.maximum((kv + 15) // 16, 0)
    for g in range(len(groups)):
        need[cu[g]] = max(need[cu[g]], prefix[g] // 16) if cu[g + 1] > cu[g] else need[cu[g]]
    width = max(1, int(need.max(initial=0)))
    blocks = int(need.sum()) + 5
    order = iter(rng.permutation(blocks).tolist())
    tables = np.full((b, width), -1, np.int32)
    for s in range(b):
        g = int(np.searchsorted(cu, s, side="right")) - 1
        lead = int(cu[g]) if g < len(groups) else s
        for c in range(int(need[s])):
            shared = g < len(groups) and s != lead and c < prefix[g] // 16
            tables[s, c] = tables[lead, c] if shared else next(order)
    kp = torch.randn((blocks, hkv, 16, d), generator=gen, device=dev).to(dtype)
    vp = torch.randn((blocks, hkv, 16, d), generator=gen, device=dev).to(dtype)
    # NaN in the slots no sequence holds
    held = np.zeros((blocks, 16), bool)
    for s in range(b):
        for c in range(int(need[s])):
            upto = kv[s] if c * 16 < kv[s] else 0
            g = int(np.searchsorted(cu, s, side="right")) - 1
            if g < len(groups) and s == cu[g]:
                upto = max(upto, prefix[g] // 16 * 16)
            held[tables[s, c], : max(0, min(16, int(upto) - c * 16))] = True
    mask = torch.from_numpy(~held).to(dev).view(blocks, 1, 16, 1)
    kp.masked_fill_(mask, math.nan)
    vp.masked_fill_(mask, math.nan)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev, torch.int32)  # noqa: E731
    return dict(q=torch.randn((hq, b, d), generator=gen, device=dev).to(dtype), kp=kp, vp=vp, tables=t(tables),
                kv=t(kv), max_kv=int(kv.max()) if b else 0, cu=t(cu), prefix=t(prefix),
                max_prefix=int(prefix.max()) if len(prefix) else 0)


def call(s, max_prefix=None, **kw):
    return ops.paged_attention_shared_prefix_gemv(
        s["q"], s["kp"], s["vp"], s["tables"], s["kv"], s["max_kv"], s["cu"], s["prefix"],
        s["max_prefix"] if max_prefix is None else max_prefix, **kw)


def check(s, **kw):
    got = call(s, **kw)
    ref64.check_attention(got, ref64.attention(s["q"], s["kp"], s["vp"], s["tables"], s["kv"]))
    assert ops.read_device_error() == (0, 0)
    return got


SHAPES = [
    ([(8, 2000)], [1, 64, 17], []),                        # beams of one request
    ([(3, 100), (1, 300), (40, 700), (2, 15)], [1, 16, 33, 200], [50, 1, 900]),  # ragged, alone in a group, < a page
    ([(5, 64), (0, 64), (7, 1)], [1], []),                 # an empty group, a prefix below a page
    ([(130, 129)], [1, 2], [3]),                           # several query tiles
    ([(2, 5000)], [700, 1], []),                           # long prefix: many splits
]


@pytest.mark.parametrize("n_rep", [1, 2, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sweep(dtype, head_dim, n_rep, cuda_device):
    for i, (groups, own, loners) in enumerate(SHAPES):
        check(make(groups, own, loners, 2 * n_rep, 2, head_dim, dtype, cuda_device, seed=i))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences_shorter_than_the_prefix_and_empty_ones(dtype, cuda_device):
    for seed, shorter in enumerate([{1: 5}, {0: 20, 2: 300}, {0: 0, 3: 0}, {3: 1}, {0: 0, 1: 0, 2: 0, 3: 0}]):
        s = make([(4, 500)], [1, 30], [], 8, 2, 128, dtype, cuda_device, seed=seed, shorter=shorter)
        got = check(s)
        for b, n in shorter.items():
            assert n > 0 or (got[:, b] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bound_below_the_prefixes_shares_less(dtype, cuda_device):
    s = make([(6, 400), (3, 90)], [5, 50], [7], 8, 4, 64, dtype, cuda_device, seed=3)
    for bound in (0, 10, 100, 399):
        check(s, max_prefix=bound)


def test_no_groups_is_plain_decode(cuda_device):
    s = make([], [], [100, 1, 33], 16, 8, 128, torch.bfloat16, cuda_device)
    check(s)
    none = make([], [], [], 16, 8, 128, torch.bfloat16, cuda_device)
    none["q"] = none["q"][:, :0]
    assert call(none).shape == (16, 0, 128)


def test_more_sequences_than_the_plan_has_threads(cuda_device):
    s = make([(700, 40), (801, 33)], [1, 20, 3], [9] * 30, 4, 2, 64, torch.bfloat16, cuda_device, seed=5)
    check(s)


def test_many_groups(cuda_device):
    s = make([(2 + i % 3, 16 * (1 + i % 5) + i % 7) for i in range(70)], [1, 20, 3], [], 8, 4, 64, torch.bfloat16,
             cuda_device, seed=6)
    check(s)


def test_skewed_contexts(cuda_device):
    # one sequence holds nearly everything behind the prefix
    s = make([(20, 320)], [1], [20000], 16, 8, 128, torch.bfloat16, cuda_device, seed=7)
    check(s)


def test_views_and_layouts(cuda_device):
    s = make([(8, 200)], [9, 40], [], 16, 8, 128, torch.bfloat16, cuda_device, seed=8)
    plain = check(s)
    wide = torch.zeros(8, 20 * 128, dtype=torch.bfloat16, device=cuda_device)
    wide[:, : 16 * 128] = s["q"].transpose(0, 1).reshape(8, -1)
    s["q"] = wide[:, : 16 * 128].view(8, 16, 128).transpose(0, 1)
    got = check(s, out_token_major=True)
    assert torch.equal(got, plain) and got.transpose(0, 1).is_contiguous()


def test_malformed_groups_are_reported(cuda_device):
    s = make([(4, 100), (4, 100)], [9], [], 16, 8, 128, torch.bfloat16, cuda_device, seed=9)
    for cu in ([0, 9, 8], [-3, 4, 8], [0, 4, 100], [5, 2, 8]):
        call(dict(s, cu=torch.tensor(cu, dtype=torch.int32, device=cuda_device)))
        assert ops.read_device_error()[0] == 1
    call(dict(s, prefix=torch.tensor([-1, 100], dtype=torch.int32, device=cuda_device)))
    assert ops.read_device_error()[0] == 1
    bad = s["tables"].clone()
    bad[0, 2] = 1 << 28
    call(dict(s, tables=bad))
    assert ops.read_device_error()[0] == 7
    call(dict(s, max_kv=s["max_kv"] - 1))  # a kv_len past the bound
    assert ops.read_device_error()[0] == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_replays_in_a_graph_and_runs_on_two_streams(dtype, cuda_device):
    s = make([(12, 900), (3, 64)], [9, 100, 31], [40], 16, 8, 128, dtype, cuda_device, seed=10)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(s)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call(s)
    for it in range(3):
        s["q"].copy_(torch.randn_like(s["q"], dtype=torch.float32).to(dtype))
        s["kv"].sub_(1)
        torch.cuda.synchronize()
        want = check(s).clone()
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [call(s) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(torch.equal(a, want) for a in again)
    del g


def test_pool_past_32_bit_offsets(cuda_device):
    num_blocks, hkv, d = 135000, 8, 128
    kp = torch.empty(num_blocks, hkv, 16, d, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.empty_like(kp)
    pages = torch.arange(num_blocks - 40, num_blocks, device=cuda_device)
    for pool in (kp, vp):
        pool[pages] = torch.randn(40, hkv, 16, d, device=cuda_device).to(torch.bfloat16)
    tables = torch.stack([pages[:20], torch.cat([pages[:15], pages[30:35]])]).int().contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    q = torch.randn(32, 2, d, device=cuda_device).to(torch.bfloat16)
    got = ops.paged_attention_shared_prefix_gemv(q, kp, vp, tables, i32(320, 301), 320, i32(0, 2), i32(240), 240)
    ref64.check_attention(got, ref64.attention(q, kp, vp, tables, i32(320, 301)))
