"""Beam selection and cache reordering on the GPU against the plain forms in 64 bits (tests/ref64.py).

Tokens and parents must be equal.  Scores: the kernel's lse carries at most 2^-22 relative error per weight
(ex2.approx), one rounding of 2^-24 per addition of at most 2^10 in a row, and the result is rounded to fp32:
|score| 2^-24 + 2^-21 + 2^-14 bounds it; the sums behind it come out near 1e-7.
"""

import math

import numpy as np
import pytest
import torch

import ref64
from femtovllm_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(logits, scores, k, finished=None, eos=-1):
    got = ops.beam_search_select(logits, scores, k, finished, eos)
    want = ref64.beam_select(logits, scores, k, finished, eos)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dead = want[2] == -math.inf
    assert torch.equal(got[2] == -math.inf, dead)
    err = (got[2].double() - want[2]).abs()[~dead]
    assert (err <= want[2].abs()[~dead] * 2.0**-24 + 2.0**-21 + 2.0**-14).all(), err.max()
    return got


def inputs(n, w, v, dtype, dev, seed=0, scale=2.5):
    gen = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn(n * w, v, generator=gen, device=dev) * scale).to(dtype)
    scores = -torch.rand(n, w, generator=gen, device=dev) * 5
    return logits, scores


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,w,k", [(1, 1, 1), (1, 4, 4), (3, 5, 10), (2, 8, 16), (7, 3, 3), (1, 32, 32), (2, 33, 40),
                                   (1, 64, 64)])
@pytest.mark.parametrize("v", [151936, 50001, 4099, 70])
def test_sweep(dtype, n, w, k, v, cuda_device):
    check(*inputs(n, w, v, dtype, cuda_device, seed=v + k), k)


@pytest.mark.parametrize("v", [1, 2, 5, 17])
def test_tiny_vocabularies(v, cuda_device):
    for w in (1, 3, 8, 40):
        k = min(64, w * v)
        check(*inputs(3, w, v, torch.float32, cuda_device, seed=v), k)
        check(*inputs(3, w, v, torch.bfloat16, cuda_device, seed=v), k)


def test_many_requests(cuda_device):
    check(*inputs(700, 4, 1000, torch.bfloat16, cuda_device), 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dtype, cuda_device):
    logits = torch.zeros(2 * 4, 40000, dtype=dtype, device=cuda_device)  # constant rows
    scores = torch.zeros(2, 4, device=cuda_device)
    check(logits, scores, 7)
    logits[:, 31000:31050] = 3.0  # a run of equal maxima across lanes and vectors
    logits[:, 100::997] = 3.0
    check(logits, scores, 40)
    scores[0, 2] = 1.0
    check(logits, scores, 64)


@pytest.mark.parametrize("order", ["ascending", "descending"])
def test_sorted_logits(order, cuda_device):
    x = torch.linspace(-20, 20, 30000, device=cuda_device)
    x = x if order == "ascending" else x.flip(0)
    logits = torch.stack([x, x * 0.5, x - 3]).contiguous()
    check(logits, torch.tensor([[0.0, -1.0, -2.0]], device=cuda_device), 33)


def test_masked_vocabularies(cuda_device):
    for dtype in DTYPES:
        low = torch.finfo(dtype).min
        for fill in (-math.inf, low):
            logits = torch.full((6, 30000), fill, dtype=dtype, device=cuda_device)
            logits[0, 29999] = 1.0             # one choice
            logits[1, [5, 7000, 123]] = torch.tensor([1.0, 2.0, 3.0], dtype=dtype, device=cuda_device)
            # row 2: nothing left; rows 3 to 5: one beam alive, nothing at all
            logits[3, 0] = 4.0
            scores = torch.tensor([[-1.0, -2.0, -0.5], [-1.0, -math.inf, -math.inf]], device=cuda_device)
            check(logits, scores, 9)


def test_values_that_are_not_numbers(cuda_device):
    logits, scores = inputs(3, 4, 20000, torch.float32, cuda_device, seed=1)
    logits[0, 77] = math.nan
    logits[1] = -math.inf
    logits[2, 19999] = math.inf
    logits[5, 0] = math.nan
    scores[1, 2] = -math.inf
    scores[1, 3] = math.nan
    logits[8:12] = math.nan  # a request without a score
    check(logits, scores, 8)


def test_logits_beyond_the_exponent_range(cuda_device):
    logits = torch.full((4, 9000), -3.4e38, device=cuda_device)
    logits[1] = 3.3e38
    logits[2, ::3] = 1000.0
    logits[3, 5] = 80.0
    check(logits, torch.zeros(2, 2, device=cuda_device), 6)


def test_first_step_and_finished_beams(cuda_device):
    for dtype in DTYPES:
        logits, scores = inputs(4, 6, 32000, dtype, cuda_device, seed=3)
        scores[:, 1:] = -math.inf
        check(logits, scores, 6)
        logits, scores = inputs(4, 6, 32000, dtype, cuda_device, seed=4)
        finished = torch.zeros(4, 6, dtype=torch.bool, device=cuda_device)
        finished[0, 0] = finished[1, 3] = finished[1, 5] = True
        finished[2] = True  # nothing live: K beyond the finished beams takes -inf candidates
        logits[6 * 2: 6 * 3] = math.nan  # and their logits are not read
        scores[1, 3] = -math.inf
        check(logits, scores, 12, finished, 2)
        check(logits, scores, 12, finished, 0)
        check(logits, scores, 12, finished, 31999)


def test_candidates_closer_than_fp32_tells(cuda_device):
    """Beams whose best candidates differ by 1e-9 to 1e-7: the order is fp64's."""
    gen = torch.Generator(device=cuda_device).manual_seed(5)
    for it in range(1, 7):
        logits = torch.randn(8, 60000, generator=gen, device=cuda_device)
        perm = torch.randperm(60000, generator=gen, device=cuda_device)
        for r in range(1, 8):
            logits[r] = logits[0][perm.roll(r)]  # the same distribution, summed in another order
            logits[r, 3] += 1e-3 * r * it        # and lse apart by next to nothing
        check(logits, torch.zeros(1, 8, device=cuda_device), 24)


def test_strided_rows(cuda_device):
    logits, scores = inputs(2, 3, 5000, torch.bfloat16, cuda_device, seed=6)
    for pad in (1, 7, 8, 120):
        wide = torch.full((6, 5000 + pad), math.nan, dtype=torch.bfloat16, device=cuda_device)
        wide[:, pad:] = logits
        check(wide[:, pad:], scores, 5)
    check(logits.t().contiguous().t(), scores, 5)  # columns first: copied


def test_select_replays_in_a_graph_and_runs_on_two_streams(cuda_device):
    logits, scores = inputs(4, 8, 50001, torch.bfloat16, cuda_device, seed=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_search_select(logits, scores, 8)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.beam_search_select(logits, scores, 8)
    for it in range(3):
        logits.copy_((torch.randn_like(logits, dtype=torch.float32) * (1 + it)).to(logits.dtype))
        torch.cuda.synchronize()
        want = check(logits, scores, 8)
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [ops.beam_search_select(logits, scores, 8) for _ in range(2)]
        torch.cuda.synchronize()
        for r in [got, *again]:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
    del g


# ------------------------------------------------------------------ reordering


def cache(n, w, kv, layers, hkv, d, dtype, dev, seed=0, spare=0, block_size=16):
    """Pools and tables of n requests of w beams: shared full pages, open pages of every row's own."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    full = [x // 16 for x in kv]
    width = max(full) + 1 + spare
    blocks = sum(full) + n * w * (1 + spare) + 2
    order = iter(rng.permutation(blocks).tolist())
    tables = np.full((n * w, width), -1, np.int32)
    for i in range(n):
        shared = [next(order) for _ in range(full[i])]
        for r in range(w):
            tables[i * w + r, : full[i]] = shared
            tables[i * w + r, full[i]: full[i] + 1 + spare] = [next(order) for _ in range(1 + spare)]
    make = lambda: torch.randn((blocks, hkv, 16, d), generator=gen, device=dev).to(dtype)  # noqa: E731
    k, v = [make() for _ in range(layers)], [make() for _ in range(layers)]
    lens = torch.from_numpy(np.repeat(np.asarray(kv, np.int32), w)).to(dev)
    return k, v, torch.from_numpy(tables).to(dev), lens


def reorder(k, v, tables, lens, parents):
    want_k, want_v = [x.clone() for x in k], [x.clone() for x in v]
    want = ref64.beam_reorder(want_k, want_v, tables, lens, parents)
    before = tables.clone()
    got = ops.beam_reorder_kvcache(k, v, tables, lens, parents)
    assert torch.equal(got, want) and torch.equal(tables, before)
    for a, b in zip([*k, *v], [*want_k, *want_v]):
        assert torch.equal(a, b)
    assert ops.read_device_error() == (0, 0)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("w", [1, 2, 3, 8, 31, 32, 33, 64])
def test_reorder_sweep(dtype, w, cuda_device):
    rng = np.random.default_rng(w)
    kv = [1, 15, 16, 17, 40, 100, 0, 32]
    k, v, tables, lens = cache(len(kv), w, kv, 2, 2, 64, dtype, cuda_device, seed=w, spare=1)
    for parents in (rng.integers(0, w, (len(kv), w)), np.zeros((len(kv), w), int), np.full((len(kv), w), w - 1),
                    np.stack([rng.permutation(w) for _ in kv]), rng.integers(0, max(1, w // 3), (len(kv), w))):
        # the rule needs every row's open pages to be its own before and after: feed the tables back
        tables = reorder(k, v, tables, lens, torch.from_numpy(parents).to(cuda_device))
        open_pages = [tables[r, int(lens[r]) // 16].item() for r in range(tables.shape[0])]
        assert len(set(open_pages)) == len(open_pages)


def test_reorder_many_layers_and_odd_heads(cuda_device):
    k, v, tables, lens = cache(2, 4, [21, 30], 67, 3, 24, torch.bfloat16, cuda_device)  # more than one launch
    reorder(k, v, tables, lens, torch.tensor([[0, 0, 1, 1], [3, 3, 3, 0]], device=cuda_device))


def test_reorder_one_pool_and_other_page_sizes(cuda_device):
    k, v, tables, lens = cache(1, 3, [20], 1, 2, 128, torch.float32, cuda_device)
    want = ref64.beam_reorder([k0 := k[0].clone()], [v[0].clone()], tables, lens, torch.tensor([[2, 2, 2]]))
    got = ops.beam_reorder_kvcache(k[0], v[0], tables, lens, torch.tensor([[2, 2, 2]], device=cuda_device))
    assert torch.equal(got, want) and torch.equal(k[0], k0)
    pool = torch.arange(4 * 2 * 8 * 64, device=cuda_device, dtype=torch.float32).view(4, 2, 8, 64)
    vp = pool + 1
    tab = torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device=cuda_device)
    kv = torch.tensor([11, 11], dtype=torch.int32, device=cuda_device)
    old = pool.clone()
    new = ops.beam_reorder_kvcache(pool, vp, tab, kv, torch.tensor([[1, 1]], device=cuda_device))
    assert new.tolist() == [[0, 2], [0, 1]]
    assert torch.equal(pool[1, :, :3], old[2, :, :3]) and torch.equal(pool[1, :, 3:], old[1, :, 3:])


def test_reorder_malformed_requests_keep_their_rows(cuda_device):
    k, v, tables, lens = cache(3, 3, [20, 40, 25], 1, 2, 64, torch.bfloat16, cuda_device)
    good = torch.tensor([[0, 0, 1], [2, 2, 2], [1, 1, 0]], device=cuda_device)
    for spoil in ("parent", "negative", "lens", "past"):
        k2, v2 = [k[0].clone()], [v[0].clone()]
        p, n = good.clone(), lens.clone()
        if spoil == "parent":
            p[1, 2] = 3
        elif spoil == "negative":
            p[1, 0] = -1
        elif spoil == "lens":
            n[4] = 39
        else:
            n[3:6] = tables.shape[1] * 16 + 1
        got = ops.beam_reorder_kvcache(k2, v2, tables, n, p)
        assert torch.equal(got[3:6], tables[3:6])
        assert ops.read_device_error() == (1, 3)
        want_k, want_v = [k[0].clone()], [v[0].clone()]
        keep = good.clone()
        keep[1] = torch.arange(3, device=cuda_device)
        want = ref64.beam_reorder(want_k, want_v, tables, lens, keep)
        assert torch.equal(got, want) and torch.equal(k2[0], want_k[0]) and torch.equal(v2[0], want_v[0])
    bad = tables.clone()
    bad[0, 1] = 1 << 20
    ops.beam_reorder_kvcache([k[0].clone()], [v[0].clone()], bad, lens, good)
    assert ops.read_device_error()[0] == 7


def test_reorder_past_32_bit_offsets(cuda_device):
    num_blocks, hkv, d = 135000, 8, 128
    kp = torch.zeros(num_blocks, hkv, 16, d, dtype=torch.bfloat16, device=cuda_device)
    vp = torch.zeros_like(kp)
    tables = torch.tensor([[5, num_blocks - 1], [5, num_blocks - 2]], dtype=torch.int32, device=cuda_device)
    kp[-1] = torch.randn(hkv, 16, d, device=cuda_device).to(torch.bfloat16)
    vp[-1] = torch.randn(hkv, 16, d, device=cuda_device).to(torch.bfloat16)
    lens = torch.tensor([25, 25], dtype=torch.int32, device=cuda_device)
    new = ops.beam_reorder_kvcache(kp, vp, tables, lens, torch.tensor([[0, 0]], device=cuda_device))
    assert torch.equal(new, tables)
    for pool in (kp, vp):
        assert torch.equal(pool[-2, :, :9], pool[-1, :, :9]) and (pool[-2, :, 9:] == 0).all()
        assert (pool[:-2] == 0).all()


# ------------------------------------------------------------------ a run of them together


@pytest.mark.parametrize("graph", [False, True])
def test_beam_search_over_a_shared_prompt(graph, cuda_device):
    """Beam search on a toy decoder: prompt prefill, then select, reorder, store, shared-prefix attention.

    Every beam's attention is compared with dense float64 attention over the tokens of its own history, so a
    page that went to the wrong beam, was copied wrongly or overwritten shows at the next step.
    """
    dev, n, w, hq, hkv, d, vocab, steps = cuda_device, 3, 5, 8, 2, 64, 500, 40
    gen = torch.Generator(device=dev).manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    emb_q, emb_k, emb_v, head = rnd(vocab, hq, d), rnd(vocab, hkv, d), rnd(vocab, hkv, d), rnd(hq * d, vocab) * 0.3
    prompt_len = [37, 64, 90]
    prompts = [torch.randint(0, vocab, (p,), generator=gen, device=dev) for p in prompt_len]
    width = (max(prompt_len) + steps + 15) // 16 + 1
    # pages: the prompt's full ones shared, the rest (open and later ones) every row's own
    tables = torch.full((n * w, width), -1, dtype=torch.int32)
    page = 0
    for i, p in enumerate(prompt_len):
        for c in range(p // 16):
            tables[i * w: (i + 1) * w, c] = page
            page += 1
        for r in range(i * w, (i + 1) * w):
            m = width - p // 16
            tables[r, p // 16:] = torch.arange(page, page + m)
            page += m
    tables = tables.to(dev)
    kp = torch.full((page, hkv, 16, d), math.nan, device=dev)
    vp = kp.clone()
    lens = torch.tensor([p for p in prompt_len for _ in range(w)], dtype=torch.int32, device=dev)
    for i, toks in enumerate(prompts):  # the prompt's keys, through row 0 of each request
        pos = torch.arange(len(toks), device=dev)
        slots = tables[i * w, pos // 16].long() * 16 + pos % 16
        ops.store_kvcache(emb_k[toks], emb_v[toks], kp, vp, slots)
    cu = torch.arange(0, n * w + 1, w, dtype=torch.int32, device=dev)
    prefix = torch.tensor(prompt_len, dtype=torch.int32, device=dev)
    scores = torch.full((n, w), -math.inf, device=dev)
    scores[:, 0] = 0.0
    first = torch.stack([emb_q[t[-1]] for t in prompts]).repeat_interleave(w, 0)  # (n w, hq, d)
    logits = (first.reshape(n * w, -1) @ head).contiguous()
    tokens = torch.zeros(n, w, dtype=torch.int64, device=dev)
    parents = torch.zeros(n, w, dtype=torch.int64, device=dev)
    attn = torch.empty(hq, n * w, d, device=dev)

    def step():
        t, p, s = ops.beam_search_select(logits, scores, w)
        new = ops.beam_reorder_kvcache(kp, vp, tables, lens, p)
        tables.copy_(new)
        tok = t.view(-1)
        ops.store_kvcache(emb_k[tok], emb_v[tok], kp, vp, ops.build_slot_mapping(lens, tables))
        lens.add_(1)
        q = emb_q[tok].transpose(0, 1)
        o = ops.paged_attention_shared_prefix_gemv(q, kp, vp, tables, lens, width * 16, cu, prefix, max(prompt_len))
        attn.copy_(o)
        logits.copy_(o.transpose(0, 1).reshape(n * w, -1) @ head)
        scores.copy_(s), tokens.copy_(t), parents.copy_(p)

    run = step
    if graph:
        saved = [x.clone() for x in (kp, vp, tables, lens, scores, logits)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        for x, y in zip((kp, vp, tables, lens, scores, logits), saved):
            x.copy_(y)
        run = g.replay
    history = [[t.tolist() for _ in range(w)] for t in prompts]
    total = [[0.0] + [-math.inf] * (w - 1) for _ in range(n)]
    prev = logits.clone()
    for it in range(steps):
        run()
        torch.cuda.synchronize()
        logp = torch.log_softmax(prev.double(), 1).view(n, w, vocab)
        history = [[history[i][parents[i, r]] + [int(tokens[i, r])] for r in range(w)] for i in range(n)]
        total = [[total[i][parents[i, r]] + float(logp[i, parents[i, r], tokens[i, r]]) for r in range(w)]
                 for i in range(n)]
        # one rounding of the running score to fp32 per step, on values below 2^10: 40 * 2^-15
        assert np.allclose(scores.cpu().numpy(), np.array(total), rtol=0, atol=steps * 2.0**-15)
        for i in range(n):
            for r in range(w):
                toks = torch.tensor(history[i][r], device=dev)
                k, v = emb_k[toks].double().transpose(0, 1), emb_v[toks].double().transpose(0, 1)
                q = emb_q[toks[-1]].double().view(hkv, hq // hkv, d)
                x = q @ k.transpose(1, 2) / math.sqrt(d)
                want = (torch.softmax(x, -1) @ v).reshape(hq, d)
                assert (attn[:, i * w + r].double() - want).abs().max() <= 1e-4, (it, i, r)  # fp32 attention's bound
        prev = logits.clone()
    assert ops.read_device_error() == (0, 0)
    if graph:
        del g
