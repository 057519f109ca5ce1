"""What a query does not see, and what a prompt is packed with, change no more than the rounding of a result."""
import math

import pytest
import torch

from tests.test_gpu_causal import check, cu_of, prompt

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from ditserve_amd import ops
    from tests.kv_reference import DEV


def attend(q, k, v, lens_q, lens_k, heads, hk, d):
    return ops.flash_attn_causal(q, k, v, ops.Segments(cu_of(lens_q), DEV), ops.Segments(cu_of(lens_k), DEV), heads, hk, d,
                                 return_lse=True)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [64, 700, 1900])
def test_hidden_scores(n, d):
    """Keys whose scores are far above all others, each hidden from the queries before it: every query within its bound,
    also where the next one's maximum moves."""
    heads, hk = 4, 2
    q, k, v = prompt([n], [n], heads, hk, d, n + d)
    k[40::97] = q[40::97, :hk * d] * 6.0
    out, lse = attend(q, k, v, [n], [n], heads, hk, d)
    check(q, k, v, [n], [n], heads, hk, d, out, lse)
    again, e = attend(q, k, v, [n], [n], heads, hk, d)
    assert torch.equal(again, out) and torch.equal(e, lse)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("x", [math.inf, -math.inf, math.nan])
def test_hidden_values_alone_and_packed(d, x):
    """A value that is not finite, in work items of 128 and of 256 queries and with few queries over many keys: the queries
    that do not see it within their bounds each time, the others infinite or NaN in its dim and within their bounds
    in all others."""
    heads, hk, key = 8, 2, 400
    lens_q, lens_k = [700, 20], [700, 1100]
    q, k, v = prompt(lens_q, lens_k, heads, hk, d, 5)
    clean = v.clone()
    for at in (key, 700 + 1090):
        v[at, 3] = x
        clean[at, 3] = 0.5
    more = 9000  # makes the launch's items large
    qm, km, vm = prompt([more], [more], heads, hk, d, 6)
    want, _ = attend(q, k, clean, lens_q, lens_k, heads, hk, d)
    results = [attend(q, k, v, lens_q, lens_k, heads, hk, d),
               attend(torch.cat([q, qm]), torch.cat([k, km]), torch.cat([v, vm]), [*lens_q, more], [*lens_k, more], heads, hk, d)]
    seen = torch.zeros((sum(lens_q), heads, d), dtype=torch.bool, device=DEV)
    seen[key:700, :heads // hk, 3] = True
    seen[700 + 1090 - 1080:, :heads // hk, 3] = True
    seen = seen.flatten(1)
    for out, lse in results:
        out, lse = out[:sum(lens_q)], lse[:, :sum(lens_q)]
        bad = out[seen].float()
        assert bool((torch.isnan(bad) if math.isnan(x) else bad == x).all())
        check(q, k, clean, lens_q, lens_k, heads, hk, d, torch.where(seen, want, out), lse)
