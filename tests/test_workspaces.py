"""Workspaces with holes: an expanded tensor has fewer bytes than elements, a strided one has others' bytes between its own. A kernel
writes in one piece from the first address on, so neither is used. What the adapters hand to the library is looked at without
a GPU."""
import pytest
import torch

from nanoengine_amd import ops

BF, FP8 = torch.bfloat16, torch.float8_e4m3fn


def holes(need):
    """Tensors of `need` bytes or more by their number of elements, but not in one piece."""
    return [torch.zeros(1, dtype=torch.uint8).expand(need + 16), torch.zeros(2 * need + 32, dtype=torch.uint8)[::2],
            torch.zeros(16, need // 8 + 16, dtype=torch.uint8)[:, 16:]]


@pytest.fixture
def calls(monkeypatch):
    """The library's calls, recorded instead of made; every tensor counts as one on the device."""
    seen = []
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: -1)  # a CPU tensor's own device number
    monkeypatch.setattr(ops, "_CURRENT_DEVICE", lambda: -1)
    monkeypatch.setattr(ops, "_launch", lambda dev, name, *args: seen.append((name, args)))
    return seen


def given(call, calls, at, **kw):
    """(address, bytes) that a call hands over at argument `at`."""
    call(**kw)
    name, args = calls.pop()
    assert not calls
    return args[at], args[at + 1]


def test_product(calls, monkeypatch):
    need = 4096
    monkeypatch.setattr(ops, "_gemm_workspace", lambda *a: need)
    a, b = torch.zeros(100, 512, dtype=FP8), torch.zeros(300, 512, dtype=FP8)
    args = dict(a=a, a_scale=torch.zeros(100, 4), b=b, b_scale=torch.zeros(3, 4))
    good = torch.zeros(need + 64, dtype=torch.uint8)
    at = (-good.data_ptr()) % 16
    assert given(ops.fp8_gemm, calls, -2, workspace=good[at:], **args) == (good.data_ptr() + at, need + 64 - at)
    for ws in holes(need):
        ptr, size = given(ops.fp8_gemm, calls, -2, workspace=ws, **args)
        assert ptr != ws.data_ptr() and size == need


@pytest.mark.gpu
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float8_e8m0fnu])
def test_product_leaves_the_bytes_between(cuda, scale_dtype):
    g = torch.Generator(device=cuda).manual_seed(0)
    a, sa = ops.act_quant(torch.randn(100, 8192, generator=g, device=cuda).to(BF), scale_dtype=scale_dtype)
    b, _ = ops.act_quant(torch.randn(300, 8192, generator=g, device=cuda).to(BF), scale_dtype=scale_dtype)
    sb = sa[:3].contiguous()
    need = ops.fp8_gemm_workspace_bytes(100, 300, 8192, scale_dtype)
    assert need > 0
    want = ops.fp8_gemm(a, sa, b, sb)
    room = torch.full((2 * need,), 0x55, dtype=torch.uint8, device=cuda)
    one = torch.full((64,), 0x55, dtype=torch.uint8, device=cuda)
    for ws in (room[::2], one[:1].expand(need), room.view(-1, 32)[:, :16]):
        assert torch.equal(ops.fp8_gemm(a, sa, b, sb, workspace=ws), want)
    assert torch.all(room == 0x55) and torch.all(one == 0x55)
