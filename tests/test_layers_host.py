"""Refusals of the block-sparse layer entry points that need no GPU: null handles and arguments give
a status and a message, never a crash."""
import ctypes as C

import pytest

import varblockspmm_b200 as vb
from varblockspmm_b200 import _lib


def refused(status, match):
    assert status == vb.INVALID_ARGUMENT
    assert match in vb.last_error()


def test_null_handles_are_refused():
    out, n = C.c_void_p(), C.c_int64()
    refused(_lib.vbsr_gated_create(None, None, 0, C.byref(out)), "null matrix")
    refused(_lib.vbsr_gated_create(None, None, 0, None), "null output")
    refused(_lib.vbsr_gated_workspace_bytes(None, 1, 0, C.byref(n)), "null plan")
    refused(_lib.vbsr_gated_forward(None, None, 1, None, None, None, None, 0, None), "null plan")
    refused(_lib.vbsr_gated_backward(None, None, None, None, None, 1, None, None, None, None, 0, None),
            "null plan")
    refused(_lib.vbsr_gated_set_values(None, None, None, None), "null plan")
    refused(_lib.vbsr_gated_check_status(None, None), "null plan")
    refused(_lib.vbsr_int8_create(None, None, None, C.byref(out)), "null matrix")
    refused(_lib.vbsr_int8_workspace_bytes(None, 1, C.byref(n)), "null plan")
    refused(_lib.vbsr_int8_execute(None, None, None, 1, None, None, 0, None), "null plan")
    refused(_lib.vbsr_int8_execute_panel(None, None, 1, None, None, 0, None), "null plan")
    refused(_lib.vbsr_int8_check_status(None, None), "null plan")
    refused(_lib.vbsr_matrix_quantize(None, None, None, None), "null matrix")
    refused(_lib.vbsr_ortho_create(None, C.byref(out)), "null matrix")
    refused(_lib.vbsr_ortho_execute(None, None, None, 5, 0.0, None, None), "null plan")
    for destroy in (_lib.vbsr_gated_destroy, _lib.vbsr_int8_destroy, _lib.vbsr_ortho_destroy):
        assert destroy(None) == vb.OK


def test_quantize_panel_arguments():
    q = _lib.vbsr_quantize_panel
    refused(q(None, 0, 1, None, None, None), "K must be positive")
    refused(q(None, 8, -1, None, None, None), "tokens")
    refused(q(None, 8, (1 << 22) + 1, None, None, None), "tokens")
    refused(q(None, 8, 1, None, None, None), "null")
    assert q(None, 8, 0, None, None, None) == vb.OK


def test_panels_that_are_not_device_tensors():
    import torch
    with pytest.raises(vb.InvalidArgument, match="CUDA"):
        vb.quantize_panel(torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2), 8)
    for K in (0, -8):
        with pytest.raises(vb.InvalidArgument, match="positive"):
            vb.quantize_panel(torch.zeros(2, 8), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2), K)


def test_matrix_of_structure_only():
    """A matrix without values needs no GPU and no values; what would read them refuses it."""
    import lm_reference as ref
    host = ref.matrix(5, 7, 3, 1)
    values = len(host.values)
    host.values = host.values[:0]
    m = vb.Matrix(host, structure_only=True)
    info = m.info()
    assert (info.block_rows, info.block_cols, info.value_count) == (5, 7, values)
    assert (info.scalar_rows, info.scalar_cols) == (host.scalar_rows(), host.scalar_cols())
    assert info.device_bytes == 0
    for call in (m.device_view, lambda: vb.Plan(m, 32)):
        with pytest.raises(vb.InvalidArgument, match="structure only"):
            call()
    refused(_lib.vbsr_matrix_quantize(m._h, None, None, None), "structure only")
    for kw in (dict(rows=(0, 2)), dict(generated_seed=1)):
        with pytest.raises(vb.InvalidArgument, match="structure_only"):
            vb.Matrix(host, structure_only=True, **kw)
    with pytest.raises(vb.InvalidArgument, match="offsets"):
        vb.Matrix(host)
    host.block_col = host.block_col + 7
    with pytest.raises(vb.InvalidArgument, match="out of range"):
        vb.Matrix(host, structure_only=True)


def test_int8_set_values_of_a_null_plan():
    refused(_lib.vbsr_int8_set_values(None, None, None, None), "null plan")


def test_int8_weights_and_scales_go_together():
    """Refused before any array is read."""
    import lm_reference as ref
    m = vb.Matrix(ref.matrix(3, 4, 2, 1), structure_only=True)
    for values, scale in ((256, None), (None, 256)):
        with pytest.raises(vb.InvalidArgument, match="null values or row_scale"):
            vb.Int8Plan(m, values, scale)
