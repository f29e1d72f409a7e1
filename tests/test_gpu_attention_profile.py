"""What a profiled call of an attention operator keeps on the device: a capture saves and restores all of it."""

import re

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["norm_rope_cache", "read", "attention"])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_a_profiled_call_keeps_its_own_inputs_alone(op, fmt, capsys):
    from mxfp4_b200 import profile

    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    profile.run_attention(op, fmt, (2, 64, 8, 128, 8192), 1)
    nbytes = int(re.search(r"bytes=(\d+)", capsys.readouterr().out)[1])
    # what the call reads and writes, that once more for the inputs' making, and 32 MB for workspaces and pages
    assert torch.cuda.max_memory_allocated() - before <= 2 * nbytes + (32 << 20)
