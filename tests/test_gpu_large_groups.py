"""Groups of more query heads than a tile holds: the window and shared-prefix operators serve them in chunks."""

import numpy as np
import pytest
import torch

from femtovllm_b200 import ops, workloads
import ref64
import test_gpu_shared_prefix as shared
from test_gpu_sharing import wide
from test_gpu_window import _decode, _prefill

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
GQA = [9, 17, 20, 32]


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_window_decode(dtype, head_dim, n_rep, cuda_device):
    """Few short sequences, and long ones whose units are cut wherever an SM's share of the tiles ends."""
    for lens, window, sinks in [([1, 40, 333, 16], 100, 5), ([3000, 777, 2048, 1, 129, 5000, 1300, 64], 1 << 30, 0),
                                ([3000, 777, 2048, 1, 129, 5000, 1300, 64] * 2, 1900, 33)]:
        b = workloads.custom(lens, np.ones(len(lens)), 4 * n_rep, 4, head_dim, dtype, seed=n_rep).materialize(cuda_device)
        _decode(b, window, sinks)


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_window_prefill(dtype, head_dim, n_rep, cuda_device):
    q_lens = np.array([1, 70, 9, 300, 2, 1])
    b = workloads.custom(q_lens + [300, 0, 90, 500, 64, 0], q_lens, 2 * n_rep, 2, head_dim, dtype,
                         seed=n_rep).materialize(cuda_device)
    for window, sinks in [(1 << 30, 0), (130, 20), (1, 0)]:
        _prefill(b, window, sinks)


@pytest.mark.parametrize("n_rep", GQA)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_prefix(dtype, head_dim, n_rep, cuda_device):
    for i, (groups, own, loners) in enumerate([([(8, 500)], [1, 64, 170], []), ([(3, 100), (1, 300), (17, 700)], [16, 200], [50]),
                                               ([(2, 5000)], [700, 1], [])]):
        s = shared.make(groups, own, loners, 2 * n_rep, 2, head_dim, dtype, cuda_device, seed=i)
        assert torch.isfinite(shared.check(s)).all()
        shared.check(wide(s))


def test_out_of_a_token_major_buffer(cuda_device):
    s = shared.make([(8, 500)], [1, 64, 170], [], 40, 2, 128, torch.bfloat16, cuda_device, seed=1)
    for t in (s, wide(s)):
        got = shared.call(t, out_token_major=True)
        assert torch.equal(got, shared.call(t)) and got.transpose(0, 1).is_contiguous()
        ref64.check_attention(got, ref64.attention(s["q"], s["kp"], s["vp"], s["tables"], s["kv"]))
    assert ops.read_device_error() == (0, 0)
