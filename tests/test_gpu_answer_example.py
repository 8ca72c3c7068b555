"""The answering example runs, its bookkeeping is right, and its logits are
those of the same decoder with exact attention, to the error of 4-bit rows."""
from __future__ import annotations

import math
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
REPO = Path(__file__).resolve().parents[1]


def test_answers(uv):
    import torch

    sys.path.insert(0, str(REPO / "examples"))
    import answer

    got = answer.main(layers=2, width=512, passages=3, tokens=5, questions=3)
    assert got["lens"] == got["used"]
    assert got["pages"] == sum(-(-n // 64) for n in got["lens"])
    refs = got["cache"].refs
    assert bool((refs[:got["pages"]] == 1).all()) and int(refs[got["pages"]:].sum()) == 0
    assert all(len(a) == 5 for a in got["answers"]) and all(1 <= k <= 4 for k in got["kept"])

    # The same tokens with exact attention.  A held row is a rotated row with a
    # relative error of 0.107 (the best 16-level uniform quantiser of a Gaussian,
    # 0.01154 of its variance), which random directions dilute through the
    # softmax; half of the logits' norm would be a wrong attention, not a rounding.
    model = got["model"]
    for i, (text, asked) in enumerate(zip(got["texts"], got["asked"])):
        ids = torch.tensor(text + asked, device="cuda")
        n = len(ids)

        def exact(layer, q, k, v):
            group = q.shape[1] // k.shape[1]
            k, v = (x.float().repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
            e = q.float().transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(q.shape[2])
            e = e.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
            return (torch.softmax(e, -1) @ v).transpose(0, 1).bfloat16()

        want = model(ids, torch.arange(n, device="cuda"), exact)[-1]
        err = float((got["logits"][i] - want).norm() / want.norm())
        assert err < 0.25, err
