"""Shared-prefix calls that are large enough to share, where tests/test_gpu_shared_prefix.py's go sequence by sequence.

A call shares its prefixes once sequences x kv heads x pages of max_kv_len (twice that at 128 dims) exceed a limit per SM
that is 256 at most, so `wide` gives a call a table and a bound beyond it; `make` and the lengths are that file's.
"""

import ctypes

import pytest
import torch

import cabi
import ref64
from femtovllm_b200 import capi, ops
import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def wide(s, limit=256):
    """The call `s` with a table and a max_kv_len that put it beyond `limit` pages an SM."""
    hkv, d = s["kp"].shape[1], s["kp"].shape[3]
    sms = torch.cuda.get_device_properties(s["q"].device).multi_processor_count
    columns = min(limit * sms // (len(s["tables"]) * hkv * (d // 64)) + 1, capi.load().fvb_max_kv_len() // 16)
    assert len(s["tables"]) * hkv * columns * (d // 64) > limit * sms
    columns = max(columns, s["tables"].shape[1])
    tables = torch.full((len(s["tables"]), columns), -1, dtype=torch.int32, device=s["tables"].device)
    tables[:, : s["tables"].shape[1]] = s["tables"]
    return dict(s, tables=tables, max_kv=16 * columns)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_groups_by_null_pointers(dtype, cuda_device):
    """Zero groups need no arrays: both may be null in the C entry, also where the call could share."""
    s = wide(shared.make([], [], [100, 1, 33, 700], 16, 8, 128, dtype, cuda_device, seed=1))
    hq, b, d = s["q"].shape
    lib, code = cabi.lib(), capi.dtype_code(dtype)
    need = lib.fvb_paged_attention_shared_prefix_workspace_size(b, hq, 8, d, s["max_kv"], 0, 0, code)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=cuda_device)
    out = torch.empty_like(s["q"])
    for max_prefix in (0, 4096):
        need = lib.fvb_paged_attention_shared_prefix_workspace_size(b, hq, 8, d, s["max_kv"], 0, max_prefix, code)
        assert need <= ws.numel()
        out.fill_(7.0)
        capi.check(lib.fvb_paged_attention_shared_prefix_decode(
            s["q"].data_ptr(), d, b * d, out.data_ptr(), d, b * d, s["kp"].data_ptr(), s["vp"].data_ptr(),
            s["kp"].shape[0], hq, 8, d, 16, b, s["tables"].data_ptr(), s["tables"].shape[1], s["kv"].data_ptr(),
            s["max_kv"], None, 0, None, max_prefix, code, ws.data_ptr(), ws.numel(),
            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "shared prefix")
        ref64.check_attention(out, ref64.attention(s["q"], s["kp"], s["vp"], s["tables"], s["kv"]))
        assert ops.read_device_error() == (0, 0)
    shared.check(s)  # and by the tensor of one entry that the Python call takes


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_groups_again_and_again(dtype, cuda_device):
    """The table of groups stands where the first tiles of keys go: it must have been read before they arrive."""
    many = [(2 + i % 3, 16 * (1 + i % 5) + i % 7) for i in range(300)]
    s = wide(shared.make(many, [1, 20, 3, 140], [], 8, 4, 64, dtype, cuda_device, seed=6))
    want = shared.check(s)
    for _ in range(30):
        assert torch.equal(shared.call(s), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_group_s_first_row_names_the_shared_pages(dtype, cuda_device):
    """Shows that these calls share: another row's entries for the shared pages are not read, its first row's are."""
    for hq, d in ((2, 64), (8, 128)):
        s = wide(shared.make([(2, 5000), (3, 90)], [700, 1], [], hq, 2, d, dtype, cuda_device, seed=4))
        want = shared.check(s)
        tables = s["tables"].clone()
        tables[1, : 5000 // 16] = -1
        tables[3:5, : 90 // 16] = 1 << 28
        assert torch.equal(shared.call(dict(s, tables=tables)), want) and ops.read_device_error() == (0, 0)
        tables[0, 7] = -1
        shared.call(dict(s, tables=tables))
        assert ops.read_device_error()[0] == 7


@pytest.mark.parametrize("dtype", DTYPES)
def test_pool_past_32_bit_offsets(dtype, cuda_device):
    num_blocks, hkv, d = 135000, 8, 128  # 2.2e9 elements a pool
    kp = torch.empty(num_blocks, hkv, 16, d, dtype=dtype, device=cuda_device)
    vp = torch.empty_like(kp)
    pages = torch.arange(num_blocks - 60, num_blocks, device=cuda_device)
    for pool in (kp, vp):
        pool[pages] = torch.randn(60, hkv, 16, d, device=cuda_device).to(dtype)
    tables = torch.stack([pages[:30], torch.cat([pages[:25], pages[40:45]])]).int().contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    s = wide(dict(q=torch.randn(32, 2, d, device=cuda_device).to(dtype), kp=kp, vp=vp, tables=tables, kv=i32(480, 461),
                  max_kv=480, cu=i32(0, 2), prefix=i32(400), max_prefix=400))
    shared.check(s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_sequences_than_a_table_holds(dtype, cuda_device):
    """1024 sequences and one more: the limit of the kernel that takes 16-bit calls."""
    for n in (1024, 1025):
        s = shared.make([(n - 30, 40)], [1, 20, 3], [9] * 30, 4, 2, 64, dtype, cuda_device, seed=5)
        shared.check(wide(s))
