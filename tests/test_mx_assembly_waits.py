"""CPU checks of the generated gfx950 assembly around the microscaled products' direct loads, as test_assembly_waits.py
makes them for the grouped products': the wait states behind a scalar base that a vector instruction wrote, and m0.
Nothing runs on a GPU."""
import shutil

import pytest

pytest.importorskip("torch")

import test_assembly_waits as waits  # noqa: E402

SOURCE = r"""
#include "ml_mx_grouped.h"
using namespace ml;
extern "C" __global__ void dwords_base(const char* const* in, float* out) {
  __shared__ __align__(1024) unsigned char lds[256];
  ring_dwords(uniform(in[threadIdx.x]), threadIdx.x * 4u, (uint32_t)(uintptr_t)(lds_void_t*)lds);
  ring_wait<0>();
  out[threadIdx.x] = ((const float*)lds)[threadIdx.x];
}
extern "C" __global__ void one_base(const char* const* in, float* out) {
  __shared__ __align__(1024) unsigned char lds[1024];
  const uint32_t off[1] = {threadIdx.x * 16u};
  ring_loads(uniform(in[threadIdx.x]), off, (uint32_t)(uintptr_t)(lds_void_t*)lds);
  ring_wait<0>();
  out[threadIdx.x] = ((const float*)lds)[threadIdx.x];
}
extern "C" __global__ void loads_between(const char* in, int n) {
  __shared__ __align__(1024) unsigned char lds[4096];
  const uint32_t at = (uint32_t)(uintptr_t)(lds_void_t*)lds, off[1] = {threadIdx.x * 16u};
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_dwords(in, off[0], at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_dwords(in + off[0], at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_loads(in, off, at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_wait<0>();
}
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if shutil.which("hipcc") is None:
        pytest.skip("no hipcc")
    source, waits.SOURCE = waits.SOURCE, SOURCE
    try:
        return waits.kernels.__wrapped__(tmp_path_factory)
    finally:
        waits.SOURCE = source


@pytest.mark.parametrize("name", ["dwords_base", "one_base"])
def test_scalar_bases_are_waited_for(kernels, name):
    code = kernels[name]
    assert any(n.startswith("v_readfirstlane") for n, _ in code)
    assert waits.wait_states(code, "v_readfirstlane", "global_load_lds") >= 5


def test_loads_declare_m0(kernels):
    waits.test_loads_declare_m0({"loads_between": kernels["loads_between"]})
