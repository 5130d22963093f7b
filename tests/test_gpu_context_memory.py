"""GPU: the token-memory operators and the index together, as an example program uses them."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_evicted_tokens_are_found_again():
    import context_memory
    r = context_memory.run(tokens=3000, steps=8, budget=256, found=32)
    assert r["flags"] == 0 and r["evicted"] == 3000 - 256
    assert torch.isfinite(r["prompt"].float()).all()
    # the tokens found carry most of what the cache had lost
    assert r["errors"]["cache and index"] < 0.5 * r["errors"]["cache"], r["errors"]
