"""CPU tests of the LM head with adapters: what its calls refuse before any device is touched."""
import ctypes

import pytest

from neuraval_b200 import native

CREATE = dict(device=0, dtype=native.DTYPE_BF16, inner=64, out=100, rows=8, adapters=4, rank=16)


def create(navlib, **over):
    h = ctypes.c_void_p()
    st = navlib.ncb_adapter_head_create(*dict(CREATE, **over).values(), ctypes.byref(h))
    return st, h


@pytest.mark.parametrize("over", [
    dict(device=-1), dict(dtype=native.DTYPE_F32), dict(dtype=7), dict(inner=0), dict(out=0),
    dict(rows=0), dict(adapters=-1), dict(rank=-1), dict(rank=0)], ids=str)
def test_create_refuses(navlib, over):
    st, h = create(navlib, **over)
    assert st == native.NCB_ERROR_INVALID_ARGUMENT and not h.value
    assert navlib.ncb_sampler_last_status() == st


@pytest.mark.parametrize("over", [dict(adapters=1025), dict(rank=129), dict(rows=1 << 17),
                                  dict(out=(1 << 24) + 1), dict(inner=(1 << 20) + 1)], ids=str)
def test_create_capacity(navlib, over):
    st, h = create(navlib, **over)
    assert st == native.NCB_ERROR_CAPACITY and not h.value


def test_calls_without_a_head(navlib):
    p = 0x1000
    assert navlib.ncb_adapter_head_create(*CREATE.values(), None) == native.NCB_ERROR_INVALID_ARGUMENT
    assert navlib.ncb_adapter_head_destroy(None) == native.NCB_ERROR_INVALID_ARGUMENT
    for st in (navlib.ncb_adapter_head_set_weight_device(None, p, 64, None),
               navlib.ncb_adapter_head_set_adapter_device(None, 0, p, 64, p, 8, 8, 1.0, None),
               navlib.ncb_adapter_head_clear_adapter_device(None, 0, None),
               navlib.ncb_adapter_head_project_device(None, p, 64, 1, p, p, 0, 100, None)):
        assert st == native.NCB_ERROR_NOT_INITIALIZED


def test_create_without_a_device_reports_it(navlib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a device is present")
    st, h = create(navlib)
    assert st in (native.NCB_ERROR_NO_DEVICE, native.NCB_ERROR_INIT_FAILED) and not h.value


def test_front_end_refuses_host_tensors():
    import torch
    from neuraval_b200.adapter_head import CudaAdapterHead
    with pytest.raises(ValueError):
        CudaAdapterHead(torch.zeros(4, 8, dtype=torch.bfloat16), max_rows=1)
    with pytest.raises(ValueError):
        CudaAdapterHead(torch.zeros(8, dtype=torch.bfloat16), max_rows=1)
