"""The decoding operators over a paged KV cache, as cases that can be timed and compared.

Five operators of a serving step, each in a plain form (elementary torch operations, ``own``
false) and as a user of ``femtovllm_b200.ops`` calls it (``own`` true):

* ``window_gemv``: decode attention with a sliding window and a few first tokens that stay
  visible (sinks);
* ``window_gemm``: the same mask for chunked prefill, single-token rows mixed in;
* ``shared_prefix``: decode attention for sequences that share a long prefix;
* ``beam_select``: the best continuations over beams x vocabulary;
* ``beam_reorder``: the KV cache and block tables follow the beams that were chosen.

Lengths, group sizes and parents come from a case's ``lens_seed`` alone, so ``work`` knows them;
contents and page numbers come from ``prepare``'s seed.
"""

import math

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEVICE = "cuda"


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------


def listed():
    return [
        # A handful of short fp32 requests: what one call costs when there is hardly any work.
        dict(name="window_gemv 4 short fp32", op="window_gemv", b=4, hq=8, hkv=2, d=64, dtype="f32", kv_lo=1,
             kv_hi=256, window=64, sinks=4, freed=False, lens_seed=1),
        # A full decode batch of a model whose layers look back 1024 tokens.
        dict(name="window_gemv 256 w1024", op="window_gemv", b=256, hq=16, hkv=8, d=128, dtype="bf16", kv_lo=512,
             kv_hi=4096, window=1024, sinks=4, freed=False, lens_seed=2),
        # Long-running sessions, eight query heads a kv head; pages behind the window were given back.
        dict(name="window_gemv 32 long gqa8", op="window_gemv", b=32, hq=64, hkv=8, d=128, dtype="bf16", kv_lo=32768,
             kv_hi=131072, window=4096, sinks=128, freed=True, lens_seed=3),
        # Chunked prefill over cached prefixes.
        dict(name="window_gemm 8 chunks w1024", op="window_gemm", b=8, hq=16, hkv=8, d=128, dtype="bf16", q_lo=128,
             q_hi=2048, p_lo=0, p_hi=4096, singles=0, window=1024, sinks=4, freed=False, lens_seed=4),
        # One engine step: decode rows and short chunks in one call, half precision, 64-wide heads.
        dict(name="window_gemm mixed f16 d64", op="window_gemm", b=24, hq=32, hkv=4, d=64, dtype="f16", q_lo=2,
             q_hi=300, p_lo=0, p_hi=1500, singles=12, window=256, sinks=0, freed=True, lens_seed=5),
        # Eight beams of one request behind a prompt that ends inside a page.
        dict(name="shared_prefix 8 beams", op="shared_prefix", b=8, groups=1, loners=0, hq=16, hkv=8, d=128,
             dtype="bf16", p_lo=2000, p_hi=2000, own_lo=1, own_hi=64, lens_seed=6),
        # 32 requests behind one 4096-token system prompt.
        dict(name="shared_prefix 32 requests", op="shared_prefix", b=32, groups=1, loners=0, hq=32, hkv=8, d=128,
             dtype="bf16", p_lo=4096, p_hi=4096, own_lo=64, own_hi=1024, lens_seed=7),
        # A busy server: four prompts of different lengths with ragged crowds behind them, and requests on their own.
        dict(name="shared_prefix 128 in 4 groups", op="shared_prefix", b=128, groups=4, loners=5, hq=32, hkv=8, d=128,
             dtype="bf16", p_lo=2048, p_hi=12288, own_lo=1, own_hi=1024, lens_seed=8),
        # One request, four beams: the latency of one step.
        dict(name="beam_select 1x4", op="beam_select", n=1, w=4, vocab=151936, k=4, dtype="bf16", done=False,
             first=False, lens_seed=9),
        # 32 requests of eight beams, twice as many candidates as beams.
        dict(name="beam_select 32x8", op="beam_select", n=32, w=8, vocab=151936, k=16, dtype="bf16", done=True,
             first=False, lens_seed=10),
        # The cache of one small request follows its beams.
        dict(name="beam_reorder 1x4", op="beam_reorder", n=1, w=4, layers=4, blocks=256, hkv=8, d=128, dtype="bf16",
             kv_lo=500, kv_hi=1000, lens_seed=11),
        # The same for 32 requests of eight beams over all layers of a model.
        dict(name="beam_reorder 32x8", op="beam_reorder", n=32, w=8, layers=28, blocks=640, hkv=8, d=128,
             dtype="bf16", kv_lo=100, kv_hi=4000, lens_seed=12),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


# Bytes and operations of the largest listed case of each operator, which no drawn one passes.
LARGEST = dict(window_gemv=(1.0e9, 4.4e9), window_gemm=(1.8e8, 1.0e11), shared_prefix=(4.0e8, 1.4e10),
               beam_select=(6.2e7, 1.2e8), beam_reorder=(1.7e8, 1.0))


def draw(rng):
    case, at = _draw(rng), "b"
    if case["op"].startswith("beam"):
        at = "n"
    while case[at] > 1 and any(w > most for w, most in zip(work(case).values(), LARGEST[case["op"]])):
        case[at] = case[at] * 3 // 4
        if case["op"] == "shared_prefix":
            case.update(groups=min(case["groups"], case["b"]), loners=min(case["loners"], (case["b"] - 1) // 4))
            case["groups"] = min(case["groups"], case["b"] - case["loners"])
        if case["op"] == "window_gemm":
            case["singles"] = min(case["singles"], case["b"])
        if case["op"] == "beam_reorder":
            case["blocks"] = case["n"] * case["w"] * 2 + 17
    return case


def _draw(rng):
    op = rng.choice(["window_gemv", "window_gemm", "shared_prefix", "beam_select", "beam_reorder"])
    case = dict(op=op, lens_seed=rng.randrange(1 << 30))
    if op in ("window_gemv", "window_gemm", "shared_prefix"):
        hkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if hkv <= 4 else [1, 2, 4, 5, 8])
        case.update(hq=hkv * group, hkv=hkv, d=rng.choice([64, 128]))
        case.update(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if op == "window_gemv":
        hi = _log(rng, 16, 65536)
        case.update(b=min(_log(rng, 1, 256), max(1, 600000 // hi)), kv_lo=max(1, _log(rng, 1, hi)), kv_hi=hi)
        case.update(window=_log(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 17, 128]), freed=rng.random() < 0.5)
    elif op == "window_gemm":
        q_hi, p_hi = _log(rng, 2, 1500), _log(rng, 1, 4000)
        b = min(_log(rng, 1, 24), max(1, 20000000 // (q_hi * (q_hi + p_hi))))
        case.update(b=b, q_lo=1 + rng.randrange(q_hi), q_hi=q_hi, p_lo=0, p_hi=p_hi, singles=rng.randrange(b + 1) // 2)
        case.update(window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 17, 128]), freed=rng.random() < 0.5)
    elif op == "shared_prefix":
        p_hi, own_hi = _log(rng, 16, 12288), _log(rng, 1, 1024)
        b = min(_log(rng, 1, 128), max(1, 1200000 // (p_hi + own_hi)))
        groups = rng.randrange(1, min(b, 6) + 1)
        case.update(b=b, groups=groups, loners=rng.randrange(0, b - groups + 1) // 4, p_lo=max(1, _log(rng, 1, p_hi)),
                    p_hi=p_hi, own_lo=1 + rng.randrange(own_hi), own_hi=own_hi)
    elif op == "beam_select":
        w = rng.choice([1, 2, 3, 4, 5, 8, 10, 16])
        k = rng.choice([w, w, 2 * w])
        vocab = rng.choice([_log(rng, 1000, 200000), 151936, 32000, 50001])
        case.update(n=max(1, min(_log(rng, 1, 32), 256 // w)), w=w, k=k, vocab=vocab)
        case.update(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), done=rng.random() < 0.4, first=rng.random() < 0.2)
    else:
        w = rng.choice([1, 2, 3, 4, 5, 8, 10, 16])
        n = max(1, min(_log(rng, 1, 32), 256 // w))
        case.update(n=n, w=w, layers=rng.choice([1, 4, 12, 28]), blocks=n * w * 2 + rng.randrange(64))
        kv_hi = _log(rng, 1, 4000)
        case.update(hkv=rng.choice([1, 2, 8]), d=rng.choice([64, 128]), dtype=rng.choice(["bf16", "f16", "f32"]))
        case.update(kv_lo=1 + rng.randrange(kv_hi), kv_hi=kv_hi)
    return case


# ----------------------------------------------------------------------------------------------
# lengths (from the case alone) and inputs (from the seed)
# ----------------------------------------------------------------------------------------------


def _between(rng, lo, hi, n):
    return rng.integers(lo, hi + 1, size=n)


def _lens(case):
    """The lengths, groups and parents of a case, as numpy arrays."""
    rng = np.random.default_rng(case["lens_seed"])
    op = case["op"]
    if op == "window_gemv":
        kv = _between(rng, case["kv_lo"], case["kv_hi"], case["b"])
        return dict(kv=kv, q=np.ones_like(kv), first=np.zeros_like(kv) + kv - 1)
    if op == "window_gemm":
        q = _between(rng, case["q_lo"], case["q_hi"], case["b"])
        q[rng.permutation(case["b"])[: case["singles"]]] = 1
        p = _between(rng, case["p_lo"], case["p_hi"], case["b"])
        return dict(kv=p + q, q=q, first=p)
    if op == "shared_prefix":
        cuts = np.sort(rng.permutation(np.arange(1, case["b"] - case["loners"]))[: case["groups"] - 1])
        cu = np.concatenate([[0], cuts, [case["b"] - case["loners"]]]).astype(np.int64)
        prefix = _between(rng, case["p_lo"], case["p_hi"], case["groups"])
        of = np.concatenate([np.repeat(prefix, np.diff(cu)), np.zeros(case["loners"], np.int64)])
        return dict(cu=cu, prefix=prefix, kv=of + _between(rng, case["own_lo"], case["own_hi"], case["b"]))
    if op == "beam_select":
        done = (rng.random((case["n"], case["w"])) < 0.2) & case["done"]
        return dict(done=done)
    # Few beams have most of the children, as after a confident step.
    weight = 1.0 / (1.0 + np.arange(case["w"]))
    parents = rng.choice(case["w"], size=(case["n"], case["w"]), p=weight / weight.sum())
    return dict(parents=parents, kv=np.repeat(_between(rng, case["kv_lo"], case["kv_hi"], case["n"]), case["w"]))


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _seen(case, first, last):
    """Pages [0, a) and [b, c) hold every key that queries first..last of a sequence see."""
    return min(_pages(case["sinks"]), last // PAGE + 1), max(0, first - case["window"] + 1) // PAGE, last // PAGE + 1


def _table(case, lens, rng):
    """(block tables, number of pool pages): pages in shuffled order, -1 where a row has none."""
    n = _pages(lens["kv"]).astype(np.int64)
    held = np.arange(n.max())[None, :] < n[:, None]
    if case["op"] == "shared_prefix":
        shared = np.concatenate([np.repeat(lens["prefix"] // PAGE, np.diff(lens["cu"])), np.zeros(case["loners"], int)])
        lead = np.concatenate([np.repeat(lens["cu"][:-1], np.diff(lens["cu"])), np.arange(lens["cu"][-1], case["b"])])
        column = np.arange(n.max())[None, :]
        common = (column < shared[:, None]) & (lead[:, None] != np.arange(case["b"])[:, None])
    else:
        common = np.zeros_like(held)
        if case["freed"]:
            for s in range(case["b"]):
                a, b, c = _seen(case, int(lens["first"][s]), int(lens["kv"][s]) - 1)
                held[s, a:max(a, b)] = False
    private = held & ~common
    blocks = int(private.sum()) + 3
    tables = np.full(held.shape, -1, np.int32)
    tables[private] = rng.permutation(blocks)[: int(private.sum())]
    if case["op"] == "shared_prefix":
        tables = np.where(common, tables[lead], tables)
    return tables, blocks


def _parents_table(case, lens, rng):
    """Block tables of beams: full pages are shared within a request, the open page of every row is its own."""
    n, w = case["n"], case["w"]
    full = (lens["kv"] // PAGE).reshape(n, w)
    width = int(full.max()) + 1
    pages = rng.permutation(case["blocks"]).astype(np.int32)
    tables = np.full((n, w, width), -1, np.int32)
    open_pages = pages[: n * w].reshape(n, w)
    for i in range(n):
        f = int(full[i, 0])
        tables[i, :, :f] = rng.choice(pages[n * w :], size=f)[None, :] if len(pages) > n * w else 0
        tables[i, :, f] = open_pages[i]
    return tables.reshape(n * w, width)


def prepare(case, seed):
    lens = _lens(case)
    rng = np.random.default_rng([seed, case["lens_seed"]])
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 1000003 + case["lens_seed"])
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)

    def on_device(x, as_type):
        return torch.from_numpy(np.ascontiguousarray(x)).to(DEVICE, as_type)

    state = dict(case)
    if case["op"] == "beam_select":
        n, w, vocab = case["n"], case["w"], case["vocab"]
        # The beams of a request agree on most of the vocabulary and differ in detail.
        common = torch.randn((n, 1, vocab), generator=gen, device=DEVICE) * 2.2
        logits = common + torch.randn((n, w, vocab), generator=gen, device=DEVICE)
        scores = -torch.rand((n, w), generator=gen, device=DEVICE) * 4 - 10
        scores = scores.sort(dim=1, descending=True).values
        if case["first"]:
            scores[:, 1:] = -math.inf
        state.update(logits=logits.reshape(n * w, vocab).to(dtype), scores=scores)
        state.update(finished=on_device(lens["done"], torch.bool) if case["done"] else None, eos=2)
        return state
    if case["op"] == "beam_reorder":
        shape = (case["layers"], case["blocks"], case["hkv"], PAGE, case["d"])
        k, v = normal(*shape), normal(*shape)
        state.update(k=k, v=v, k_pools=list(k.unbind(0)), v_pools=list(v.unbind(0)))
        state.update(tables=on_device(_parents_table(case, lens, rng), torch.int32))
        state.update(kv_lens=on_device(lens["kv"], torch.int32), parents=on_device(lens["parents"], torch.int64))
        return state
    tables, blocks = _table(case, lens, rng)
    tokens = case["b"] if case["op"] != "window_gemm" else int(lens["q"].sum())
    shape = (blocks, case["hkv"], PAGE, case["d"])
    state.update(q=normal(case["hq"], tokens, case["d"]), k=normal(*shape), v=normal(*shape))
    state.update(tables=on_device(tables, torch.int32), kv_lens=on_device(lens["kv"], torch.int32))
    state.update(max_kv=int(lens["kv"].max()))
    if case["op"] == "window_gemm":
        cu = np.concatenate([[0], np.cumsum(lens["q"])])
        positions = np.concatenate([np.arange(f, f + n) for f, n in zip(lens["first"], lens["q"])])
        state.update(cu=on_device(cu, torch.int32), positions=on_device(positions, torch.int32))
        state.update(max_q=int(lens["q"].max()))
    if case["op"] == "shared_prefix":
        state.update(cu=on_device(lens["cu"], torch.int32), prefix=on_device(lens["prefix"], torch.int32))
        state.update(max_prefix=int(lens["prefix"].max()))
    return state


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------


def _gather(pool, tables, keys):
    """(B, L, Hkv, D) in 32 bits: the rows of keys (B, L) of every sequence; keys without a page read page 0."""
    page = tables.gather(1, (keys // PAGE).clamp(0, tables.shape[1] - 1)).clamp(min=0).long()
    return pool[page, :, keys % PAGE].float()


def _softmax_v(scores, seen, v, formula):
    """softmax over the last axis where `seen`, times v; a row that sees nothing gives zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.einsum(formula, p / torch.where(total == 0, torch.ones_like(total), total), v)


def _plain_decode(q, k_pool, v_pool, tables, keys, seen):
    """(Hq, B, D): decode attention over keys (B, L), of which `seen` (B, L) count."""
    hq, b, d = q.shape
    k, v = _gather(k_pool, tables, keys), _gather(v_pool, tables, keys)
    hkv = k.shape[2]
    scores = torch.einsum("hgbd,blhd->bhgl", q.float().view(hkv, hq // hkv, b, d), k) * d**-0.5
    out = _softmax_v(scores, seen[:, None, None, :], v, "bhgl,blhd->hgbd")
    return out.reshape(hq, b, d).to(q.dtype)


def _plain_window_gemv(s):
    last = s["kv_lens"].long()[:, None] - 1
    sink = torch.arange(s["sinks"], device=DEVICE)[None, :].expand(last.shape[0], -1)
    near = last - torch.arange(min(s["window"], s["max_kv"]), device=DEVICE)[None, :]
    seen = torch.cat([sink <= last, near >= s["sinks"]], 1)
    return _plain_decode(s["q"], s["k"], s["v"], s["tables"], torch.cat([sink, near], 1).clamp(min=0), seen)


def _plain_window_gemm(s):
    q, cu, d = s["q"], s["cu"].long(), s["d"]
    hq, hkv = s["hq"], s["hkv"]
    step = torch.arange(s["max_q"], device=DEVICE)
    here = cu[:-1, None] + step[None, :]  # token of (sequence, row); rows past a chunk repeat its last token
    live = here < cu[1:, None]
    here = torch.minimum(here, cu[1:, None] - 1)
    keys = torch.arange(s["max_kv"], device=DEVICE)[None, :].expand(here.shape[0], -1)
    k, v = _gather(s["k"], s["tables"], keys), _gather(s["v"], s["tables"], keys)
    at = s["positions"].long()[here][:, :, None]
    key = keys[:, None, :]
    seen = (key <= at) & (key < s["kv_lens"].long()[:, None, None]) & ((at - key < s["window"]) | (key < s["sinks"]))
    rows = q.float()[:, here].view(hkv, hq // hkv, *here.shape, d)
    scores = torch.einsum("hgbqd,blhd->bhgql", rows, k) * d**-0.5
    out = _softmax_v(scores, seen[:, None, None], v, "bhgql,blhd->hgbqd").reshape(hq, *here.shape, d)
    return out[:, live].to(q.dtype)


def _plain_shared_prefix(s):
    keys = torch.arange(s["max_kv"], device=DEVICE)[None, :].expand(s["b"], -1)
    return _plain_decode(s["q"], s["k"], s["v"], s["tables"], keys, keys < s["kv_lens"].long()[:, None])


def _plain_beam_select(s):
    n, w, vocab = s["n"], s["w"], s["vocab"]
    x = s["logits"].double()  # two candidates may lie closer together than 32 bits tell apart
    top = x.amax(1, keepdim=True)
    x = x - (top + torch.exp(x - top).sum(1, keepdim=True).log())
    total = s["scores"].double().view(n * w, 1) + x
    if s["finished"] is not None:
        finished = s["finished"].view(n * w, 1)
        total = total.masked_fill(finished, -math.inf)
        total[:, s["eos"]] = torch.where(finished[:, 0], s["scores"].double().view(-1), total[:, s["eos"]])
    best, at = torch.sort(total.view(n, w * vocab), dim=1, descending=True, stable=True)
    best, at = best[:, : s["k"]], at[:, : s["k"]]
    return at % vocab, at // vocab, best.float()


def _plain_beam_reorder(s):
    n, w = s["n"], s["w"]
    parents = s["parents"]
    row = torch.arange(w, device=DEVICE)
    same = parents[:, :, None] == parents[:, None, :]
    surplus = (same & (row[None, :] < row[:, None])).any(2)  # not its parent's first child
    idle = ~(parents[:, :, None] == row).any(1)  # rows without a child: as many as surplus ones
    match = (surplus.cumsum(1)[:, :, None] == idle.cumsum(1)[:, None, :]) & surplus[:, :, None] & idle[:, None, :]
    donor = torch.where(surplus, match.int().argmax(2), parents)
    base = torch.arange(n, device=DEVICE)[:, None] * w
    parent_row, donor_row = (base + parents).view(-1), (base + donor).view(-1)
    full, fill = s["kv_lens"].long() // PAGE, s["kv_lens"].long() % PAGE
    column = torch.arange(s["tables"].shape[1], device=DEVICE)[None, :]
    tables = torch.where(column < full[:, None], s["tables"][parent_row], s["tables"][donor_row])
    moved = surplus.view(-1) & (fill > 0)
    at = full[moved][:, None]
    source = s["tables"][parent_row[moved]].gather(1, at)[:, 0].long()
    target = tables[moved].gather(1, at)[:, 0].long()
    filled = (torch.arange(PAGE, device=DEVICE)[None, :] < fill[moved][:, None])[None, :, None, :, None]
    s["k"][:, target] = torch.where(filled, s["k"][:, source], s["k"][:, target])
    s["v"][:, target] = torch.where(filled, s["v"][:, source], s["v"][:, target])
    return tables, s["k"], s["v"]


# ----------------------------------------------------------------------------------------------
# the framework's operators, and one pass
# ----------------------------------------------------------------------------------------------


def _ops():
    import sys
    from pathlib import Path

    package = str(Path.cwd() / "nano-vllm-practice_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from femtovllm_b200 import ops

    return ops


def _own(s):
    ops = _ops()
    if s["op"] == "window_gemv":
        return ops.paged_attention_window_gemv(s["q"], s["k"], s["v"], s["tables"], s["kv_lens"], s["max_kv"],
                                               s["window"], s["sinks"])
    if s["op"] == "window_gemm":
        return ops.paged_attention_window_gemm(s["q"], s["k"], s["v"], s["cu"], s["max_q"], s["tables"],
                                               s["kv_lens"], s["positions"], s["window"], s["sinks"])
    if s["op"] == "shared_prefix":
        return ops.paged_attention_shared_prefix_gemv(s["q"], s["k"], s["v"], s["tables"], s["kv_lens"], s["max_kv"],
                                                      s["cu"], s["prefix"], s["max_prefix"])
    if s["op"] == "beam_select":
        return ops.beam_search_select(s["logits"], s["scores"], s["k"], s["finished"], s["eos"])
    tables = ops.beam_reorder_kvcache(s["k_pools"], s["v_pools"], s["tables"], s["kv_lens"], s["parents"])
    return tables, s["k"], s["v"]


def run(state):
    if own:
        return _own(state)
    return {
        "window_gemv": _plain_window_gemv,
        "window_gemm": _plain_window_gemm,
        "shared_prefix": _plain_shared_prefix,
        "beam_select": _plain_beam_select,
        "beam_reorder": _plain_beam_reorder,
    }[state["op"]](state)


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without, and its answer in 64 bits
# ----------------------------------------------------------------------------------------------


def work(case):
    lens, es = _lens(case), BYTES[case["dtype"]]
    op = case["op"]
    if op == "beam_select":
        rows = int((~lens["done"]).sum())
        return dict(bytes=rows * case["vocab"] * es + case["n"] * (4 * case["w"] + 20 * case["k"]),
                    flops=4 * rows * case["vocab"])
    if op == "beam_reorder":
        parents, fill = lens["parents"], (lens["kv"] % PAGE).reshape(case["n"], case["w"])
        children = (parents[:, :, None] == np.arange(case["w"])).sum(1)
        surplus = np.maximum(children - 1, 0).sum(1)
        tokens = int((surplus * fill[:, 0]).sum())
        tables = 2 * 4 * int((lens["kv"] // PAGE + 1).sum())
        return dict(bytes=2 * 2 * tokens * case["hkv"] * case["d"] * es * case["layers"] + tables + 8 * parents.size,
                    flops=0)
    row = case["hkv"] * case["d"] * es * 2  # K and V of one token
    kv, b = lens["kv"], case["b"]
    if op == "shared_prefix":
        shared = lens["prefix"] // PAGE * PAGE
        sizes = np.diff(lens["cu"])
        keys = int(kv.sum() - (shared * (sizes - 1)).sum())
        pairs, tokens, entries = int(kv.sum()), b, keys // PAGE + 2 * b
    else:
        first, q = lens["first"], lens["q"]
        tokens, pairs, keys, entries = int(q.sum()), 0, 0, b
        for s in range(b):
            at = np.arange(first[s], first[s] + q[s])
            near = np.minimum(at + 1, case["window"])
            sinks = np.minimum(np.maximum(at - case["window"] + 1, 0), case["sinks"])
            pairs += int((near + sinks).sum())
            keys += int(min(kv[s], kv[s] - max(0, first[s] - case["window"] + 1) + sinks[0]))
        entries += keys // PAGE
    qo = 2 * case["hq"] * tokens * case["d"] * es
    return dict(bytes=keys * row + qo + 4 * entries + 4 * b, flops=4 * case["hq"] * case["d"] * pairs)


def exact(case, seed):
    op = case["op"]
    if op == "beam_reorder":  # copies: nothing is computed
        return None
    s = prepare(case, seed)
    if op == "beam_select":
        tokens, beams, scores = [], [], []
        for i in range(case["n"]):
            x = s["logits"][i * case["w"] : (i + 1) * case["w"]].double()
            total = s["scores"][i].double()[:, None] + torch.log_softmax(x, 1)
            if s["finished"] is not None:
                for j in torch.nonzero(s["finished"][i])[:, 0].tolist():
                    total[j] = -math.inf
                    total[j, s["eos"]] = s["scores"][i, j].double()
            flat = total.reshape(-1)
            least = torch.topk(flat, case["k"]).values[-1]
            at = torch.nonzero(flat >= least)[:, 0].cpu().numpy()
            value = flat[torch.from_numpy(at).to(flat.device)].cpu().numpy()
            at = at[np.lexsort((at, -value))][: case["k"]]
            tokens.append(at % case["vocab"])
            beams.append(at // case["vocab"])
            scores.append(flat.cpu().numpy()[at])
        return np.stack(tokens), np.stack(beams), np.stack(scores)
    lens = _lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    cost = float(work(case)["flops"]) if op != "window_gemm" else 4.0 * hq * d * float((lens["q"] * lens["kv"]).sum())
    if cost > 2e13:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    start = 0
    for i in range(case["b"]):
        n = int(lens["q"][i]) if op == "window_gemm" else 1
        length = int(lens["kv"][i])
        page = s["tables"][i, : _pages(length)].long().clamp(min=0)
        k = s["k"][page].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :length].double()
        v = s["v"][page].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :length].double()
        x = s["q"][:, start : start + n].double().reshape(hkv, -1, d) @ k.transpose(1, 2) / math.sqrt(d)
        x = x.view(hkv, hq // hkv, n, length)
        if op != "shared_prefix":
            at = torch.arange(length - n, length, device=DEVICE)[:, None]
            key = torch.arange(length, device=DEVICE)[None, :]
            x = torch.where((key <= at) & ((key > at - case["window"]) | (key < case["sinks"])), x, -math.inf)
        out[:, start : start + n] = (torch.softmax(x, -1).view(hkv, -1, length) @ v).view(hq, n, d)
        start += n
    return out
