"""The 8-bit cache's and packed attention's entry points without a device:
null plans and bad arguments are refused before any CUDA call, and a pager of
8-bit pools keeps its tables like the others."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    import molot_b200
    return molot_b200


def test_null_and_bad_arguments(lib):
    L = lib.library()
    assert L.molot_f8b_plan_create(None) == lib.ERR_INVALID
    assert L.molot_packed_plan_create(None) == lib.ERR_INVALID
    L.molot_f8b_plan_destroy(None)
    L.molot_packed_plan_destroy(None)
    lens = np.array([5], np.int32)
    assert L.molot_f8b_plan_build(None, 1, 4, 2, 64, lens.ctypes.data, None, None, None, 0,
                                  None) == lib.ERR_INVALID
    assert L.molot_packed_plan_build(None, 1, 4, 2, 64, lens.ctypes.data, None, None, 0,
                                     None) == lib.ERR_INVALID
    assert L.molot_f8b_write(None, None, None, None, 0, 0, 0, None) == lib.ERR_INVALID
    assert L.molot_f8b_decode(None, None, None, None, None, 0, 0, 1.0, 0.0, None, None,
                              None) == lib.ERR_INVALID
    assert L.molot_f8b_evict(None, None, None, 8, 4, None, None) == lib.ERR_INVALID
    assert L.molot_f8b_evict(None, None, None, 0, 0, None, None) == lib.ERR_INVALID
    assert L.molot_f8b_evict(None, None, None, 4, 5, None, None) == lib.ERR_INVALID
    assert L.molot_f8b_check(None, None) == lib.ERR_INVALID
    assert L.molot_packed_attend(None, None, None, None, None, None, 1, 0, 0, 0, 1.0, 0.0, None,
                                 None) == lib.ERR_INVALID
    assert L.molot_packed_check(None, None) == lib.ERR_INVALID
    assert lib.last_error()


def test_pager_of_f8b_pools(lib):
    p = lib.Pager(0, 2, 128, 16, 4, 2, 3, dtype="f8b")
    s = p.add(20)
    bt, lens = p.tables([s])
    assert p.free_pages() == 2 and lens.tolist() == [20] and bt[0, :2].tolist() == [0, 1]
    with pytest.raises(lib.MolotError):  # tables only: no pools
        p.layer_blocks(0)
    p.close()
    with pytest.raises(lib.MolotError) as e:
        lib.Pager(0, 2, 96, 16, 4, 2, 3, dtype="f8b")
    assert e.value.status == lib.ERR_INVALID
    assert lib.library().molot_pager_layer_blocks(None, 0, None, None, None) == lib.ERR_INVALID


def test_other_caches_refuse_f8b(lib):
    h = ctypes.c_void_p()
    assert lib.library().molot_kv_create_ex(1, 2, 128, 16, lib.KV_F8B,
                                            ctypes.byref(h)) == lib.ERR_INVALID
    assert lib.library().molot_paged_plan_set_kv_dtype(None, lib.KV_F8B) == lib.ERR_INVALID
    with pytest.raises(ValueError):
        lib.KVCache(1, 2, 128, 16, dtype="f8b")


def test_cpp_wrappers_compile(tmp_path):
    src = tmp_path / "f8.cc"
    src.write_text('''
#include "molot_b200/attn.hpp"
void serve(molot_b200::Pager& pager, const int* lens, const int* bt, const void* x, void* o,
           int* kept) {
  molot_b200::F8Plan plan;
  plan.build(1, 8, 2, 64, lens);
  molot_f8b_layer l = pager.f8_layer(0, bt, 16);
  plan.write(l, x, x, MOLOT_ACT_BF16, 12 * 64, 12 * 64);
  plan.decode(l, x, o, MOLOT_ACT_BF16, 0.125f, 30.f, nullptr, nullptr, l.weight);
  plan.evict(l, l, 8, 4, kept);
  plan.sync();
  molot_b200::PackedPlan packed;
  packed.build(1, 8, 2, 64, lens);
  packed.attend(x, x, x, o, MOLOT_ACT_F16, 0.125f);
  packed.sync();
}
''')
    cxx = os.environ.get("CXX", "g++")
    subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-c", str(src), "-I",
                    os.path.join(ROOT, "include"), "-o", str(tmp_path / "f8.o")], check=True)
