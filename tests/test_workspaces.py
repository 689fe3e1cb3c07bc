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


@pytest.fixture
def old_calls(calls, monkeypatch):
    """The same for the adapters that ask torch for devices and streams."""
    monkeypatch.setattr(ops, "_check_cuda", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops._lib, "call", lambda name, *args: calls.append((name, args)))
    return calls


def mla_inputs(row):
    return dict(q=torch.zeros(4, 16, 576, dtype=BF), k_cache=torch.zeros(2, 64, 1, row, dtype=torch.uint8),
                indices=torch.zeros(4, 128, dtype=torch.int32), sm_scale=1.0, num_splits=2)


@pytest.mark.parametrize("name,row,at", [("sparse_mla_decode", 656, -3), ("sparse_mla_decode_fp4", 400, -2)])
def test_attention_takes_its_own(old_calls, monkeypatch, name, row, at):
    need = 4096
    monkeypatch.setattr(ops, "sparse_mla_workspace_bytes", lambda *a: need)
    call, args = getattr(ops, name), mla_inputs(row)
    good = torch.zeros(need + 16, dtype=torch.uint8)
    good = good[(-good.data_ptr()) % 16:]
    assert given(call, old_calls, at, workspace=good, **args) == (good.data_ptr(), good.numel())
    for ws in holes(need):
        ptr, size = given(call, old_calls, at, workspace=ws, **args)
        assert ptr != ws.data_ptr() and size == need


def refusing():
    i32, f32, u8 = torch.int32, torch.float32, torch.uint8
    rows, idx = torch.zeros(3, 4096), torch.zeros(3, 2048, dtype=i32)
    lens = torch.zeros(3, dtype=i32)
    tables = torch.zeros(3, 64, dtype=i32)
    yield "topk_transform", -3, dict(scores=rows, seq_lens=lens, page_tables=tables, out_page_indices=idx, page_size=64, top_k=2048)
    yield "topk_transform_raw", -3, dict(scores=rows, seq_lens=lens, out_indices=idx, top_k=2048)
    yield "indexer_select", -3, dict(logits=rows, context_lens=lens, out_indices=idx, top_k=2048)
    yield "topk_transform_ragged", -3, dict(scores=rows, seq_lens=lens, row_starts=lens, offsets=lens, out_indices=idx, top_k=2048)
    q = torch.zeros(3, 64, 128, dtype=u8)
    yield "indexer_topk", -4, dict(q_fp8=q[:, None], kv_cache=torch.zeros(2, 64 * 132, dtype=u8), weights=torch.zeros(3, 64),
                                   context_lens=lens, block_tables=tables, max_context_len=4096, top_k=2048, out_physical=idx)
    yield "mqa_topk", -3, dict(q_fp8=q, kv_fp8=torch.zeros(4096, 128, dtype=u8), kv_scale=torch.zeros(4096),
                               weights=torch.zeros(3, 64), ks=lens, ke=lens, max_len=4096, out=idx)
    cu = torch.tensor([0, 3], dtype=i32)
    yield "sparse_mla_prefill_paged", -3, dict(
        q=torch.zeros(3, 16, 576, dtype=BF), k_cache=torch.zeros(2, 64, 1, 656, dtype=u8), block_table=tables[:1], cu_seqlens_q=cu,
        cu_seqlens_k=cu, total_k=3, fresh=torch.zeros(3, 576, dtype=BF), indices=idx, sm_scale=1.0)


@pytest.mark.parametrize("name,at,args", refusing(), ids=[r[0] for r in refusing()])
def test_the_others_refuse(old_calls, name, at, args):
    need, call = 1 << 20, getattr(ops, name)
    good = torch.zeros(need, dtype=torch.uint8)
    assert given(call, old_calls, at, workspace=good, **args) == (good.data_ptr(), need)
    for ws in holes(need):
        with pytest.raises(RuntimeError, match="contiguous"):
            call(workspace=ws, **args)
    assert not old_calls


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
