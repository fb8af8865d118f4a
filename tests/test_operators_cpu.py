"""Refusals of the linear cross entropy and the embedding that need no GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch


class _Handle:
    """Stands in for a DeviceContext in calls that are refused before the library is entered."""

    device = 0
    handle = None


def test_linear_ce_defaults(ob):
    from orda_b200 import _abi

    o = _abi.OrdaLinearCeOptions()
    ob.load_library().orda_linear_ce_options_default(C.byref(o))
    assert (o.ignore_index, o.label_smoothing, o.reduction, o.global_non_ignore, o.piece_bytes) == (-100, 0.0, 0, 0, 0)


def test_linear_ce_null_arguments(ob):
    from orda_b200 import _abi

    buf = _abi.err_buf()
    rc = ob.load_library().orda_linear_cross_entropy_device(None, None, None, None, 0, None, None, None, buf, len(buf))
    assert rc == _abi.ORDA_ERR_INVALID and b"null" in buf.value


@pytest.mark.parametrize("change,what", [
    ({"labels": torch.zeros(4, dtype=torch.int32)}, "int64"),
    ({"labels": torch.zeros(8, dtype=torch.int64)[::2]}, "contiguous"),
    ({"labels": torch.zeros(2, 2, dtype=torch.int64)}, "1-D"),
    ({"hidden": torch.zeros(4, dtype=torch.bfloat16)}, "2-D"),
    ({"out": {"grad": torch.zeros(4, 8)}}, "unknown outputs"),
    ({}, "context's device"),
])
def test_linear_ce_python_refusals(ob, change, what):
    from orda_b200.device import linear_cross_entropy_device

    args = {"hidden": torch.zeros(4, 8, dtype=torch.bfloat16), "weight": torch.zeros(6, 8, dtype=torch.bfloat16),
            "labels": torch.zeros(4, dtype=torch.int64)}
    args.update(change)
    with pytest.raises(ValueError, match=what):
        linear_cross_entropy_device(_Handle(), **args)


def test_embedding_null_arguments(ob):
    from orda_b200 import _abi

    buf = _abi.err_buf()
    lib = ob.load_library()
    assert lib.orda_embedding_device(None, None, None, 0, 1.0, None, None, buf, len(buf)) == _abi.ORDA_ERR_INVALID
    assert b"null" in buf.value
    buf = _abi.err_buf()
    rc = lib.orda_embedding_grad_device(None, None, None, 0, 1.0, 0, 0, None, 0, None, buf, len(buf))
    assert rc == _abi.ORDA_ERR_INVALID and b"null" in buf.value


def test_embedding_python_refusals(ob):
    from orda_b200.device import embedding_device, embedding_grad_device

    table, ids = torch.zeros(6, 8), torch.zeros(4, dtype=torch.int64)
    for args, what in [((table[0], ids), "2-D"), ((table.T, ids), "unit column stride"), ((table, ids.int()), "int64"),
                       ((table, torch.zeros(8, dtype=torch.int64)[::2]), "contiguous"), ((table, ids), "device")]:
        with pytest.raises(ValueError, match=what):
            embedding_device(_Handle(), *args)
    g = torch.zeros(4, 8)
    for args, what in [((g, ids.int(), 6), "int64"), ((g, ids, 6), "device")]:
        with pytest.raises(ValueError, match=what):
            embedding_grad_device(_Handle(), *args)
