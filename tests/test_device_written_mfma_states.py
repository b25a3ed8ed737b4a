"""The wait states behind the matrix instructions that the prompt attention writes as instructions, taken from the compiler: as many
as it puts itself between such a product and the first instruction that reads the result."""
import re
import subprocess

from inferno_amd.build import COMMON_FLAGS, CSRC, hipcc
from tests import test_device_written_mfma as base

PRODUCT = """
#include <hip/hip_runtime.h>
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float acc_t __attribute__((ext_vector_type(%d)));
__global__ void product(const bf16x8_t* a, float* out) {
  const acc_t c = __builtin_amdgcn_mfma_f32_%s_bf16(a[0], a[threadIdx.x], acc_t{}, 0, 0, 0);
  for (int i = 0; i < %d; ++i) out[64 * i + threadIdx.x] = 2.0f * c[i];
}
"""


def _assembly(source, out):
    subprocess.run([hipcc(), *COMMON_FLAGS, "--cuda-device-only", "-S", str(source), "-o", str(out)], check=True, capture_output=True)
    return out.read_text()


def states_of_the_compiler(tmp_path, shape, values):
    source = tmp_path / f"product_{shape}.hip"
    source.write_text(PRODUCT % (values, shape, values))
    lines = [l.split(";")[0].strip() for l in _assembly(source, tmp_path / f"{shape}.s").splitlines()]
    at = next(i for i, l in enumerate(lines) if l.startswith("v_mfma"))
    result = base._registers(re.split(r",\s*(?![^\[]*\])", lines[at].partition(" ")[2])[0])
    states = 0
    for line in lines[at + 1:]:
        op, _, rest = line.partition(" ")
        if not line or line.startswith("."):
            continue
        if op.startswith("v_") and base._registers(rest) & result:
            return states
        states += int(rest) + 1 if op == "s_nop" else 1
    raise AssertionError("no reader")


def test_prompt_attention_keeps_the_states_of_the_compiler(tmp_path, monkeypatch):
    states = max(states_of_the_compiler(tmp_path, shape, values) for shape, values in (("32x32x16", 16), ("16x16x32", 4)))
    assert states >= 12
    monkeypatch.setattr(base, "RESULT_STATES", states)
    product = ("v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]", True)
    reader = [("v_accvgpr_read_b32 v8, a15", False), ("s_endpgm", False)]
    assert base.too_close([product, (f"s_nop {states - 2}", False), *reader])
    assert not base.too_close([product, (f"s_nop {states - 1}", False), *reader])
    kernels = {n: l for n, l in base._functions(_assembly(CSRC / "window_prefill.hip", tmp_path / "prompts.s")).items()
               if any(hand and t.startswith("v_mfma") for t, hand in l)}
    assert len(kernels) == 9
    for name, lines in kernels.items():
        assert not base.too_close(lines), name
