"""Beam selection's order where fp32 sums cannot tell: it is that of the scores in 64 bits (tests/ref64.py).

Tokens and parents must be equal; the oracle's own sums are off by less than 1e-13, and the true scores compared here
lie further apart than that, or are equal in every bit because their rows are.
"""

import math

import pytest
import torch

import ref64
from femtovllm_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(logits, scores, k, finished=None, eos=-1):
    tokens, parents, got = ops.beam_search_select(logits, scores, k, finished, eos)
    want = ref64.beam_select(logits, scores, k, finished, eos)
    assert torch.equal(tokens, want[0]) and torch.equal(parents, want[1])
    return got, want[2]


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_differ_in_one_small_logit(dtype, cuda_device):
    """The beam with less weight in its tail scores more everywhere, by 1e-12 to 1e-9: it comes first, token by token."""
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    for low in (-14.0, -12.0, -10.0, -8.0):
        for heavy in (0, 1):
            row = (torch.randn(50001, generator=gen, device=cuda_device) * 2).clamp(min=-7.0).to(dtype)
            logits = row.repeat(2, 1)
            logits[:, 40000] = low - 1
            logits[heavy, 40000] = low
            lse = torch.logsumexp(logits.double(), 1)
            assert 1e-12 < (lse[heavy] - lse[1 - heavy]).item() < 1e-7
            for k in (1, 2, 7, 40):
                check(logits, torch.zeros(1, 2, device=cuda_device), k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_copies(dtype, cuda_device):
    """Equal in every bit: the lower beam comes first.  (The oracle's sums of copies differ in their last bits, so the
    order here is that of the logits themselves, which copies share.)"""
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    row = (torch.randn(3, 1, 30011, generator=gen, device=cuda_device) * 2).to(dtype)
    logits = row.expand(3, 5, 30011).reshape(15, -1).contiguous()
    tokens, parents, _ = ops.beam_search_select(logits, torch.zeros(3, 5, device=cuda_device), 20)
    at = torch.sort(logits.view(3, -1).double(), dim=1, descending=True, stable=True).indices[:, :20]
    assert torch.equal(tokens, at % 30011) and torch.equal(parents, at // 30011)


@pytest.mark.parametrize("k", [4, 32, 64])
@pytest.mark.parametrize("extra", [1, 3, 200])
def test_rivals_behind_equal_logits_at_the_cut(extra, k, cuda_device):
    """One beam has more equal largest logits than are selected; the other's, next in line, score 1e-10 to 1e-8 more.

    Its row holds the same logits in another order, so that both sums are one and the same but for fp32's roundings, and
    one of them is a little smaller.  With 200 equal logits a beam the candidates are too many to be ranked at once.
    """
    gen = torch.Generator(device=cuda_device).manual_seed(k + extra)
    v, n = 60000, 24
    logits = torch.randn(n, 1, v, generator=gen, device=cuda_device).repeat(1, 2, 1)
    for i in range(n):
        logits[i, 0, torch.randperm(v, generator=gen, device=cuda_device)[: k + extra]] = 5.0
        logits[i, 1] = logits[i, 0][torch.randperm(v, generator=gen, device=cuda_device)]
        small = int((logits[i, 1] - 2.0).abs().argmin())  # holds about 7e-5 of the weight
        logits[i, 1, small] -= 10.0 ** (-6 + i % 8 / 4)
    logits = logits.view(2 * n, v)
    lse = torch.logsumexp(logits.double(), 1).view(n, 2)
    assert (lse[:, 0] - lse[:, 1] > 1e-11).all() and (lse[:, 0] - lse[:, 1] < 1e-5).all()
    scores = torch.zeros(n, 2, device=cuda_device)
    check(logits, scores, k)
    order = torch.arange(2 * n, device=cuda_device).view(n, 2).flip(1).reshape(-1)
    check(logits[order].contiguous(), scores, k)



def _plateau(n, v, low, dtype, dev):
    """Rows of one low value with a zero among every 1024: each warp's sum is relative to zero from its start."""
    x = torch.full((n, v), low, dtype=dtype, device=dev)
    x[:, 5::1024] = 0.0
    return x


@pytest.mark.parametrize("low", [(-3.40625, -2.15625), (-2.15625, -3.40625), (-1.3125, -4.6875), (-7.25, -9.5)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_equal_logits(dtype, low, cuda_device):
    """Thousands of equal terms take the same rounding each time they are added: the sums of two such rows err most.

    150 requests of two beams whose best scores are -2e-6 to 2e-6 apart, in rows of one part, where the sums are longest.
    """
    n, v = 150, 131000
    logits = torch.stack([_plateau(n, v, low[0], dtype, cuda_device), _plateau(n, v, low[1], dtype, cuda_device)], 1)
    logits = logits.view(2 * n, v)
    lse = torch.logsumexp(logits[:2].double(), 1)
    scores = torch.zeros(n, 2, dtype=torch.float64, device=cuda_device)
    scores[:, 1] = lse[1] - lse[0] + torch.linspace(-2e-6, 2e-6, n, dtype=torch.float64, device=cuda_device)
    check(logits, scores.float(), 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_by_the_sums_error(dtype, cuda_device):
    """Every selected score within 1.3e-6, the derived error of a sum, and its own rounding."""
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    cases = [_plateau(4, 200000, low, dtype, cuda_device) for low in (-3.40625, -2.15625, -16.0, -12.0, -0.5)]
    cases += [(torch.randn(4, v, generator=gen, device=cuda_device) * s).to(dtype)
              for v, s in ((151936, 2.5), (151936, 0.0), (50001, 12.0), (1000, 5.0), (400000, 1.0))]
    cases.append(torch.linspace(-30, 30, 4 * 100000, device=cuda_device).view(4, -1).to(dtype))
    for logits in cases:
        got, want = check(logits, torch.zeros(4, 1, device=cuda_device), 8)
        assert ((got.double() - want).abs() <= 1.3e-6 + want.abs() * 2.0**-24).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_copies_among_rows_that_nearly_are(dtype, cuda_device):
    """Twins and beams that differ from them in one small logit only, in every order: each kind by its own score."""
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    row = (torch.randn(40001, generator=gen, device=cuda_device) * 2).clamp(min=-7.0).to(dtype)
    kinds = torch.tensor([[0, 1, 0, 2, 1, 0], [2, 2, 1, 1, 0, 0], [1, 0, 2, 0, 2, 2], [0, 0, 0, 0, 0, 1]])
    logits = row.repeat(24, 1)
    for r, kind in enumerate(kinds.view(-1).tolist()):
        logits[r, 33333] = -9.0 - kind  # the higher the kind, the less weight in the tail: it scores more
    tokens, parents, _ = ops.beam_search_select(logits, torch.zeros(4, 6, device=cuda_device), 30)
    value, at = torch.sort(row.double(), descending=True, stable=True)
    assert (value[:30] > -7.0).all()
    for n in range(4):
        # by value, then by kind, then by beam, then by token
        want = sorted(((-value[i].item(), -kinds[n, w].item(), w, at[i].item()) for i in range(31) for w in range(6)))[:30]
        assert list(zip(parents[n].tolist(), tokens[n].tolist())) == [(w, i) for _, _, w, i in want]
