"""Registers of the kernels over 8-bit keys and values, read from the built libraries (no GPU)."""
import pytest

from llm_inference_lab_amd.kernels import build
from test_kernel_registers import SIMD_REGISTERS, kernels, library


@pytest.mark.parametrize("d,kernel,waves,least", [(64, "e4m3_staged_kernelIDF16b", 4, 3), (128, "e4m3_staged_kernelIDF16b", 2, 3),
                                                  (64, "e4m3_staged_kernelIf", 3, 2), (128, "e4m3_staged_kernelIf", 2, 2), (64, "e4m3_split", 2, 3),
                                                  (128, "e4m3_split", 2, 3)])
def test_waves_a_simd_holds(d, kernel, waves, least):
    taken = {name: v for name, v in kernels(library(lambda: build.e4m3_attention_library(d))).items() if kernel in name}
    assert len(taken) >= least
    for name, (registers, spilled) in taken.items():
        assert spilled == 0 and SIMD_REGISTERS // (-(-registers // 8) * 8) >= waves, (name, registers, spilled)
