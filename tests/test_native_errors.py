"""Refusals of the native modules whose message carries a number: they raise (and leave the process alive)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from gollek_b200.native import cuda_ext, host_ext


def test_unknown_ggml_type_raises():
    with pytest.raises(RuntimeError, match="ggml type 99"):
        host_ext().gguf_dequantize(torch.zeros(64, dtype=torch.uint8), 99, 32)


def test_gemm_workspace_refusal_raises():
    """The check comes before any launch, so tensors without storage do; no GPU is needed."""
    with FakeTensorMode():
        a, b, out = (torch.empty(*s, dtype=torch.bfloat16, device="cuda") for s in ((8, 128), (256, 128), (8, 256)))
        with pytest.raises(RuntimeError, match="split-K 2 needs an fp32 workspace of 4096"):
            cuda_ext().gemm_bf16(out, a, b, None, 0, 128, None, 0, 2, None)
