"""CPU checks of the generated gfx950 assembly around the device helpers that the compiler's
hazard pass does not look into (it treats inline assembly as one opaque instruction): small
kernels that put a helper right behind its operands' writers are compiled, and the wait
states between them are counted.  Nothing runs on a GPU."""
import re
import shutil
import subprocess

import pytest

pytest.importorskip("torch")

from mask_loss_amd import _build

SOURCE = r"""
#include "ml_grouped.h"
using namespace ml;
template <int DT>
__device__ void pack(const u32x4_t* in, uint32_t* out) {
  const int i = threadIdx.x;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  acc = GMma<DT>::mma(in[i], in[64 + i], acc);
  out[i] = GMma<DT>::pack(acc[0], acc[1]);
}
extern "C" __global__ void pack_f16(const u32x4_t* in, uint32_t* out) { pack<ML_F16>(in, out); }
extern "C" __global__ void pack_bf16(const u32x4_t* in, uint32_t* out) { pack<ML_BF16>(in, out); }
extern "C" __global__ void load_base(const char* const* in, float* out) {
  __shared__ __align__(1024) unsigned char lds[2048];
  const uint32_t off[2] = {threadIdx.x * 16u, threadIdx.x * 16u + 1024u};
  ring_loads(uniform(in[threadIdx.x]), off, (uint32_t)(uintptr_t)(lds_void_t*)lds);
  ring_wait<0>();
  out[threadIdx.x] = ((const float*)lds)[threadIdx.x];
}
extern "C" __global__ void loads_between(const char* in, int n) {
  __shared__ __align__(1024) unsigned char lds[4096];
  const uint32_t at = (uint32_t)(uintptr_t)(lds_void_t*)lds, off[2] = {threadIdx.x * 16u, threadIdx.x * 16u + 1024u};
  const uint32_t off4[4] = {off[0], off[1], off[0], off[1]};
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_loads(in, off, at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_loads(in, off4, at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_load(in + off[0], at);
  __builtin_amdgcn_s_sendmsg(1, n);
  ring_wait<0>();
}
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Instructions (name, operands) of each kernel above."""
    if shutil.which("hipcc") is None:
        pytest.skip("no hipcc")
    at = tmp_path_factory.mktemp("asm")
    (at / "probe.hip").write_text(SOURCE)
    subprocess.run(["hipcc", *_build.HIPCC_FLAGS, "-I" + _build.CSRC, "--cuda-device-only", "-S", str(at / "probe.hip"),
                    "-o", str(at / "probe.s")], check=True, capture_output=True, timeout=300)
    out, cur = {}, None
    for line in (at / "probe.s").read_text().splitlines():
        line = line.split(";")[0].strip()
        if re.fullmatch(r"\w+:", line):
            cur = out.setdefault(line[:-1], [])
        elif cur is not None and line and not line.startswith("."):
            name, _, rest = line.partition(" ")
            name, _, tabbed = name.partition("\t")
            cur.append((name, [o.strip() for o in (tabbed + rest).split(",")]))
            if name == "s_endpgm":
                cur = None
    return out


def registers(operand):
    """{("v", 2), ("v", 3)} of "v[2:3]"."""
    out = set()
    for kind, lo, hi, one in re.findall(r"\b([vsa])(?:\[(\d+):(\d+)\]|(\d+)\b)", operand):
        out |= {(kind, i) for i in (range(int(lo), int(hi) + 1) if lo else [int(one)])}
    return out


def wait_states(code, writer, reader):
    """Wait states between the last instruction that `writer` matches and the first one behind it that
    `reader` matches and that reads a register it wrote."""
    at = max(i for i, (name, _) in enumerate(code) if re.match(writer, name))
    wrote, states = registers(code[at][1][0]), 0
    for name, ops in code[at + 1:]:
        if re.match(reader, name) and any(registers(o) & wrote for o in ops):
            return states
        states += int(ops[0], 0) + 1 if name == "s_nop" else 1
    raise AssertionError("no reader in %r" % code)


def test_matrix_results_are_waited_for(kernels):
    """The rounding of a matrix instruction's result comes as late behind it as the compiler puts an
    instruction of its own (bfloat16's conversion)."""
    own = wait_states(kernels["pack_bf16"], "v_mfma", "v_")
    assert own > 0
    assert wait_states(kernels["pack_f16"], "v_mfma", "v_") >= own


def test_scalar_bases_are_waited_for(kernels):
    """A load's scalar base that a vector instruction wrote: five wait states."""
    code = kernels["load_base"]
    assert any(name.startswith("v_readfirstlane") for name, _ in code)
    assert wait_states(code, "v_readfirstlane", "global_load_lds") >= 5


def test_loads_declare_m0(kernels):
    """A value that the compiler keeps in m0 (a message's) is set again behind loads that use m0."""
    held, messages = None, []
    for name, ops in kernels["loads_between"]:
        if ops[0] == "m0":
            held = ops[1]
        elif name == "s_sendmsg":
            messages.append(held)
    assert len(messages) == 4 and len(set(messages)) == 1
