"""The serving example: pieces and decodes over the paged cache give what the whole sequence gives."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("budget", [64, 2000])
def test_pieces_agree_with_the_whole_sequence(dtype, quant, budget, cuda_device):
    import torch

    from mxflashattn_b200 import _lib

    sys.path.insert(0, os.path.join(REPO, "examples"))
    try:
        import chunked_serving
    finally:
        sys.path.pop(0)
    _lib.read_error_flags()
    steps, tokens, _, diff = chunked_serving.serve(dtype=torch.bfloat16 if dtype == "bf16" else torch.float16,
                                                   quant=quant, budget=budget)
    assert tokens == 700 + 37 + 1300 + 5 + 4 * 8 and steps >= 8
    # both sides round P and the output once to 16 bits: 2 * (2^-8 or 2^-11) * |values of about 4| at most
    assert diff <= 2 * 4 * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -11)
    assert _lib.read_error_flags() == 0


@pytest.mark.gpu
def test_the_example_runs_as_a_command(cuda_device):
    out = subprocess.run([sys.executable, os.path.join(REPO, "examples", "chunked_serving.py"), "--budget", "300"],
                         capture_output=True, text=True, timeout=280)
    assert out.returncode == 0, out.stderr[-800:]
    assert "largest difference" in out.stdout
