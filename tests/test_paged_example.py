"""The paged operators run together (examples/beam_search.py): beam scores against a recomputation from scratch, which has
no cache, no pages and no beams. Bound: 2e-3 relative, four layers of fp32 attention over fp16 keys and values, each
step's log-softmax to 1e-5, summed over the steps."""
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("requests,beams,steps", [(1, 1, 3), (3, 4, 20), (5, 3, 40)])
def test_beam_search_scores(requests, beams, steps):
    import beam_search as ex
    from gptoss_b200 import capi
    model, r = ex.Model(3), np.random.RandomState(requests)
    prompts = [r.randint(0, ex.VOCAB, r.randint(1, 150)) for _ in range(requests)]
    scores, tokens = ex.search(capi.load(), model, prompts, beams, steps, compact_every=5)
    s = scores.cpu().numpy()
    assert np.isfinite(s).all() and (np.diff(s, axis=1) <= 0).all()
    for i, p in enumerate(prompts):
        seen = {tuple(t.tolist()) for t in tokens[i]}
        assert len(seen) == beams
        for b in range(beams):
            want = ex.plain_score(model, p, tokens[i, b].cpu().numpy())
            assert abs(want - s[i, b]) <= 2e-3 * max(1.0, abs(want)), (i, b, want, s[i, b])
