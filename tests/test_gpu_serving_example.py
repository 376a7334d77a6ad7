"""The serving example's attention block: prompts followed by single tokens
give the outputs of one pass over the whole sequences.  Both read the same
4-bit keys and values; what differs is the attention's kernel (weights
rounded to FP16 against another reference maximum), so its MXINT8 copy may
differ by one step where a value lies near the middle of two codes."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))


def test_tokens_one_by_one_equal_the_whole_prompt(hrb):
    from serve_attention import AttentionBlock
    lengths, prompts = [75, 60, 49], [69, 54, 43]
    gen = torch.Generator(device="cuda").manual_seed(3)
    xs = [torch.randn(n, 960, device="cuda", generator=gen) for n in lengths]
    whole = AttentionBlock(hrb, requests=3, max_kv=80)
    want = whole.step(torch.cat(xs), lengths).split(lengths)
    block = AttentionBlock(hrb, requests=3, max_kv=80)
    got = [[y] for y in block.step(torch.cat([x[:p] for x, p in zip(xs, prompts)]), prompts).split(prompts)]
    for i in range(6):
        y = block.step(torch.cat([x[p + i:p + i + 1] for x, p in zip(xs, prompts)]), [1, 1, 1])
        for g, row in zip(got, y.split(1)):
            g.append(row)
    for w, g in zip(want, got):
        w, g = w.double().cpu().numpy(), torch.cat(g).double().cpu().numpy()
        # One step of MXINT8 is at most 2^-6 of its block's largest value; of
        # 960 addends only those near a middle move, so a row is within 2^-6 of
        # its own size.
        off = np.linalg.norm(g - w, axis=1) / np.linalg.norm(w, axis=1)
        assert off.max() <= 2.0 ** -6, off.max()
