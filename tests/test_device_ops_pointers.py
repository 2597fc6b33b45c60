"""Pointers that the operators on caller-owned device buffers refuse on the host: ones that a kernel could
not read (a misaligned int32 or f32), and outputs over what every CTA still reads."""
import pytest
from test_device_ops_args import P, cross, kb, lora, refused


@pytest.mark.parametrize("field", ["key_mask", "q_starts", "k_starts"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_cross_misaligned(field, off):
    refused(kb.cross_attention_f16, cross(**{field: P + off}), "4-byte aligned")


@pytest.mark.parametrize("field", ["scales", "seg_starts", "seg_adapters"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_lora_misaligned(field, off):
    refused(kb.lora_matmul_f16, lora(**{field: P + off}), "4-byte aligned")


def test_cross_outputs_over_inputs():
    refused(kb.cross_attention_f16, cross(q=P, out=P, k=3 * P, v=4 * P, out_stride=264), "same stride")
    refused(kb.cross_attention_f16, cross(q=P, out=2 * P, k=2 * P), "may not be k or v")
    refused(kb.cross_attention_f16, cross(q=P, out=2 * P, v=2 * P), "may not be k or v")
