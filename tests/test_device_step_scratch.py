"""Registers of the norm and sampling kernels in the gfx950 code: a row of a norm stays in them, and of the sampling kernels
the one for more than 4,608 sub-chunks (vocabularies past 294,905) alone has some of its 33 a thread in scratch memory."""
import re

from tests.test_device_barriers import _device_code


def _scratch(source, tmp_path):
    asm = _device_code(source, tmp_path)
    return {k: int(n) for k, n in re.findall(r"\.amdhsa_kernel (\S+).*?\.amdhsa_private_segment_fixed_size (\d+)", asm, re.S)}


def test_rows_of_a_norm_stay_in_registers(tmp_path):
    sizes = _scratch("norm_residual.hip", tmp_path)
    assert len(sizes) == 16 and not any(sizes.values()), {k: n for k, n in sizes.items() if n}


def test_sampling_kernels_with_scratch(tmp_path):
    sizes = _scratch("sample.hip", tmp_path)
    assert len(sizes) == 10
    spilling = {k for k, n in sizes.items() if n}
    assert spilling <= {k for k in sizes if re.search(r"sample_pick_kernelILb[01]ELi33E", k)}, spilling
    assert max(sizes.values()) <= 336
