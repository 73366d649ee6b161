"""The Qwen decoder's reserved flag bits are refused (on the CPU: before any tensor is looked at)."""
import ctypes as C

import pytest


@pytest.mark.parametrize("flags", [4, 7, 1 << 31, 0xFFFFFFFF])
@pytest.mark.parametrize("from_bundle", [False, True])
def test_unknown_flags_are_refused(itts, tmp_path, flags, from_bundle):
    lib, q = itts._lib, C.c_void_p(1)
    config = itts._QwenConfig(1, flags)
    if from_bundle:
        import numpy as np

        path = itts.write_mit2_bundle(tmp_path / "qwen.mit2", {"qwen.model.norm.weight": np.ones(1024, np.float32)}, single_file=True)
        bundle = itts.Bundle(path, require_model=False)
        status = lib.itts_qwen_create_from_bundle(bundle._b, C.byref(config), C.byref(q))
        bundle.close()
    else:
        status = lib.itts_qwen_create((itts._Tensor * 1)(), 0, C.byref(config), C.byref(q))
    assert status == -1 and not q.value
    assert lib.itts_qwen_last_error(None) == b"Unknown Qwen flag"


@pytest.mark.parametrize("flags", [0, 1, 2, 3])
def test_known_flags_reach_the_tensors(itts, flags):
    q = C.c_void_p()
    assert itts._lib.itts_qwen_create((itts._Tensor * 1)(), 0, C.byref(itts._QwenConfig(1, flags)), C.byref(q)) == -2
    assert itts._lib.itts_qwen_last_error(None).startswith(b"Missing tensor")
