"""The example's serving form gives what its training form gives, adapters included.

Both quantise the block's input and the hidden; the serving form's adapters read
the restored codes, and its output is codes again.  Each quantisation adds 0.9%
to 1.5% of a normal row's norm, of which at most four meet: 6%.
"""

from __future__ import annotations

import importlib.util

import pytest
import torch

import anima_flat_b200 as afb
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 77, 512])
def test_served_block_is_the_trained_one(tokens, cuda_dev):
    spec = importlib.util.spec_from_file_location("int8_lora_block", ROOT / "examples" / "int8_lora_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    p = example.make_block(256, 512, 16, cuda_dev, g)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    trained = dict(p, lora_up=afb.LoRA(p["lora_up"].a, 0.3 * randn(512, 16)), lora_down=afb.LoRA(p["lora_down"].a, 0.3 * randn(256, 16)))
    h, z = randn(1, tokens, 256), randn(1, tokens, 256)
    with torch.no_grad():
        for block in (p, trained):
            want, stream = example.run_block(block, h, z)
            q, s, served = example.serve_block(block, *afb.rowquant_int8(h), z)
            for got, ref in ((afb.int8_restore(q, s), want), (served, stream)):
                assert got.shape == ref.shape
                assert (got.float() - ref.float()).norm() <= 0.06 * ref.float().norm()
        plain = example.run_block(p, h, z)[0].float()
        assert (plain - want.float()).norm() >= 0.12 * want.float().norm()  # the adapters change the block
