"""cached_attention over pages of more than 2^31 elements (4.6 GB of keys and as much of values), in every kind of block."""
import ctypes

import numpy as np
import pytest

from cinn_amd import _lib
from cinn_amd.common import BFloat16, DefaultAMDGPUTarget, Int
from cinn_amd.frontend import Computation, NetBuilder

from test_gpu_cached_attention import Case
from typed_inputs import assert_within

pytestmark = pytest.mark.gpu

PAGES = 140000


@pytest.mark.parametrize("layout", ["row_head", "head_row"])
def test_pages_behind_2_31_elements(gpu, layout):
    for tokens, heads in ((1, 8), (3, 64), (30, 16), (50, 32)):
        case = Case("bfloat16", [1000, 70, 3], tokens, heads, 8, 128, 16, layout=layout)
        held = case.data["k_pages"].shape[0]
        far = np.random.default_rng(tokens).permutation(PAGES)[:held]
        far[case.data["table"][0, :3]] = [PAGES - 1, 131072, 131071]  # the last, and either side of 2^31 elements
        b = NetBuilder("far")
        inputs = [b.create_input(Int(32) if x.dtype == np.int32 else BFloat16(),
                                 [PAGES, *x.shape[1:]] if "pages" in n else list(x.shape), n) for n, x in case.data.items()]
        o = b.cached_attention(*inputs, page_layout=layout)
        comp = Computation.build_and_compile(DefaultAMDGPUTarget(), b, outputs=[o])
        for name, x in case.data.items():
            if "pages" not in name:
                comp.get_tensor(name).from_numpy(far[x].astype(np.int32) if name == "table" else x)
                continue
            at = comp.get_tensor(name).device_ptr
            for page, to in zip(np.ascontiguousarray(x), far):
                _lib.check_hip(_lib.load().cinn_hip_memcpy_h2d(ctypes.c_void_p(at + int(to) * page.nbytes), page.ctypes.data_as(ctypes.c_void_p),
                                                               ctypes.c_size_t(page.nbytes), None), "cinn_hip_memcpy_h2d")
        comp.execute()
        want, bound = case.reference()
        assert_within(comp.get_tensor(o.id).numpy(), want, bound, "bfloat16")
