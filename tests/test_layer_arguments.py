"""What a layer's calls cannot use is refused while the layer is made, or before the residual stream is updated: a caller that mends
its arguments and calls again adds nothing twice."""
import pytest
import torch

from nanoengine_amd import ops, projections, synth

BF, U8 = torch.bfloat16, torch.uint8


def weights(D=256, rank=128, H=2, nope=64, v=32):
    shapes = dict(norm=(D,), a=(rank + 704, D), q_norm=(rank,), kv_norm=(512,), q=(H * (nope + 64), rank), k_up=(H, nope, 512),
                  v_up=(H, 512, v), o=(D, H * v), idx_q=(8192, rank), idx_gate=(64, D), idx_norm=(128,), idx_bias=(128,))
    return {k: torch.zeros(s) for k, s in shapes.items()}


@pytest.mark.parametrize("kw", [dict(D=264), dict(rank=136), dict(v=4)])
def test_depths_that_no_product_takes(kw):
    with pytest.raises(ValueError, match="multiple of 16"):
        projections.MlaProjections(**weights(**kw), cos_sin_cache=torch.zeros(8, 64))


@pytest.mark.parametrize("kw", [dict(cos_sin_cache=torch.zeros(8, 32)), dict(cos_sin_cache=torch.zeros(8, 64).double())])
def test_tables_that_no_rotation_takes(kw):
    with pytest.raises(RuntimeError, match="cos_sin_cache"):
        projections.MlaProjections(**weights(), **kw)


def test_arguments_before_the_residual(monkeypatch):
    layer = projections.MlaProjections(**weights(), cos_sin_cache=torch.zeros(8, 64))
    reached = []
    monkeypatch.setattr(ops, "rms_norm_quant", lambda *a, **kw: reached.append(1) or ops._fail("reached"))
    T = 3
    good = dict(hidden=torch.zeros(T, 256, dtype=BF), residual=torch.zeros(T, 256, dtype=BF), positions=torch.zeros(T, dtype=torch.int64),
                slot_mapping=torch.zeros(T, dtype=torch.int64), kv_cache=torch.zeros(2, 64, 1, 656, dtype=U8),
                indexer_cache=torch.zeros(2, synth.IDX_PAGE_BYTES, dtype=U8))
    with pytest.raises(RuntimeError, match="GPU only"):
        layer.inputs(**good)
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: 0)
    for name, bad in (("positions", good["positions"][:2]), ("positions", good["positions"].float()), ("slot_mapping", good["slot_mapping"][:2]),
                      ("slot_mapping", good["slot_mapping"].float()), ("kv_cache", torch.zeros(2, 64, 1, 400, dtype=U8)),
                      ("indexer_cache", torch.zeros(2, 64 * 68, dtype=U8))):
        with pytest.raises(RuntimeError) as e:
            layer.inputs(**{**good, name: bad})
        assert "reached" not in str(e.value), name
    assert not reached
    with pytest.raises(RuntimeError, match="reached"):
        layer.inputs(**good)


def test_no_tokens_ask_for_nothing():
    layer = projections.MlaProjections(**weights(), cos_sin_cache=torch.zeros(8, 64))
    hidden = torch.zeros(0, 256, dtype=BF)
    for positions in (torch.zeros(0, dtype=torch.int64), torch.zeros(5, dtype=torch.int64), None):
        q_idx, w, q, stream = layer.inputs(hidden, None, positions, positions, None, None)
        assert q_idx.shape == (0, 64, 128) and w.shape == (0, 64) and q.shape == (0, 2, 576) and stream is hidden
