"""Registers of the kernels over 8-bit keys and values at every head size that is built beforehand, read from the libraries (no GPU)."""
import pytest

from llm_inference_lab_amd.kernels import build
from test_kernel_registers import SIMD_REGISTERS, kernels, library

# waves a SIMD that each kernel is to hold, by the first head size from which on it is so many
WAVES = {"e4m3_staged_kernelIDF16bLi2ELi4E": {16: 4, 80: 2}, "e4m3_staged_kernelIDF16bLi2ELi2E": {16: 4, 80: 3, 112: 2, 128: 3},
         "e4m3_staged_kernelIDF16bLi4ELi1E": {16: 4, 80: 3, 112: 2, 128: 3}, "e4m3_staged_kernelIf": {16: 3, 80: 2},
         "e4m3_split_kernelIDF16bLi1E": {16: 4, 80: 3, 128: 2, 256: 1}, "e4m3_split_kernelIDF16bLi2E": {16: 3, 64: 2},
         "e4m3_split_kernelIf": {16: 3, 80: 2, 256: 1}, "e4m3_merge": {16: 4}}


@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 256])
def test_nothing_is_spilled(d):
    taken = kernels(library(lambda: build.e4m3_attention_library(d)))
    names = [k for k in WAVES if not (d > 128 and ("staged" in k or "Li2E" in k))]
    assert len(taken) == (11 if d <= 128 else 5)                # (nothing that no call reaches)
    for name, (registers, spilled) in taken.items():
        kernel = [k for k in names if k in name]
        assert len(kernel) == 1, name
        waves = max(WAVES[kernel[0]].items(), key=lambda at: at[0] if at[0] <= d else -1)[1]
        assert spilled == 0 and SIMD_REGISTERS // (-(-registers // 8) * 8) >= waves, (name, registers, spilled)
