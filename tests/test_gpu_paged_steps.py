"""Steps of a server whose sequences draft a number of tokens of their own, with the rule for the lengths as the integration guide has it."""
import os
import re

import numpy as np
import pytest
import torch

from my_nn_engine_b200 import ops

GUIDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")


def rule():
    """What a step takes off the lengths again, as an expression of draft_counts, counts, accepted and K."""
    with open(GUIDE) as f:
        return re.search(r"`lengths -= ([^`]+)`", f.read()).group(1)


def test_lengths_behind_a_step_are_those_of_the_kept_tokens():
    """The last token and the accepted drafts stay; a sequence without new tokens keeps its length."""
    draft_counts, counts, accepted, K = np.array([3, 3, 1, 0, 0, 2]), np.array([4, 4, 2, 1, 0, 3]), np.array([3, 0, 1, 0, 0, 1]), 3
    before = np.array([10, 20, 30, 40, 50, 60])
    after = before + counts - eval(rule(), {}, dict(draft_counts=draft_counts, counts=counts, accepted=accepted, K=K))
    assert (after == before + np.where(counts > 0, 1 + accepted, 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,page", [("bf16", 64, 16), ("f16", 128, 24), ("f32", 40, 10)])
def test_steps_of_ragged_drafts(dt, D, page):
    """Four steps: drafts of 0 to K tokens, idle sequences, rejected tokens that the next step overwrites.  Behind each step the cache holds the keys and values of the kept tokens."""
    from test_gpu_paged import DT, cache, close_append, close_attention, draft_inputs, host, same, want_append, want_attention, want_verify
    rng = np.random.default_rng(D)
    B, H, G, K, V = 6, 8, 2, 3, 500
    S, start = K + 1, [10, 50, 33, 0, 97, 5]
    k, v, table = cache(rng, [n + 4 * S for n in start], G, D, page, dt)
    cos, sin = (torch.from_numpy(f(rng.uniform(0, 7, (200, D // 2)))).float().cuda() for f in (np.cos, np.sin))
    at = lambda t, b, j: host(t)[int(table[b, j // page]), :, j % page]
    kept = [[(at(k, b, j), at(v, b, j)) for j in range(n)] for b, n in enumerate(start)]
    lengths = torch.tensor(start, dtype=torch.int32, device="cuda")
    for step in range(4):
        draft_counts = torch.from_numpy(rng.integers(0, K + 1, B)).int().cuda()
        counts = draft_counts + 1
        draft_counts[(step + 2) % B], counts[(step + 2) % B] = 0, 0  # an idle one
        target, near, tokens, accept, sample = draft_inputs(rng, B, K, V, "f32")
        lengths += counts
        n, c, d = lengths.tolist(), counts.tolist(), draft_counts.tolist()
        proj = torch.from_numpy(rng.standard_normal((B, S, (H + 2 * G) * D))).to("cuda", DT[dt])
        wq, wk, wv = want_append(proj, n, c, table, k, v, H, cos, sin, True, False, 1e-6)
        q = ops.paged_rotary_append(proj, lengths, table, k, v, H, cos, sin, counts=counts)
        close_append(q, wq, dt)
        close_append(k, wk, dt)
        assert same(v, wv)
        want, mass = want_attention(q, k, v, table, n, c, D ** -0.5)
        close_attention(ops.paged_attention(q, k, v, table, lengths, D ** -0.5, counts=counts), want, mass, dt)
        out, accepted = ops.verify_draft(target, tokens, accept, sample, near, draft_counts)
        w, m = want_verify(target, near, tokens, d, accept, sample)
        assert np.array_equal(out.cpu().numpy(), w) and np.array_equal(accepted.cpu().numpy(), m)
        lengths -= eval(rule(), {}, dict(draft_counts=draft_counts, counts=counts, accepted=accepted, K=K))
        for b in range(B):
            if c[b]:
                first = n[b] - c[b]
                kept[b] += [(at(k, b, j), at(v, b, j)) for j in range(first, first + 1 + m[b])]
        assert lengths.tolist() == [len(x) for x in kept]
        for b, rows in enumerate(kept):
            for j, (a, e) in enumerate(rows):
                assert same(at(k, b, j), a) and same(at(v, b, j), e)
    assert any(len(x) > n + 4 for x, n in zip(kept, start))
