"""Refusals whose text holds numbers."""
import subprocess
import sys

import pytest

from vllm_sly_radiance_b200.ops import _ext


@pytest.mark.skipif(not _ext.available(), reason="the extension is not built")
def test_refusal_with_a_number_in_its_text():
    """A misaligned output is an exception, in a process of its own: text with numbers ended the process."""
    code = """if True:
        import torch
        from vllm_sly_radiance_b200.ops._ext import ext
        x, s = torch.zeros(2, 256, dtype=torch.bfloat16), torch.empty(2)
        q = torch.empty(513, dtype=torch.uint8)[1:].view(torch.float8_e4m3fn).view(2, 256)
        try:
            ext().quant_fp8_rows(x, q, s)
        except RuntimeError as e:
            assert "8-byte aligned" in str(e), e
            print("refused")
    """
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "refused", (r.returncode, r.stderr[-500:])
