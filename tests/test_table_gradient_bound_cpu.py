"""The bound on the table's gradient is tight enough: with the sums over far parts left out, doubled or turned round, the
gradient is beyond it in every case."""
import pytest
import torch

from table_gradient_bound import CASES, expected, far_parts, inputs


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_a_mistake_in_the_far_sums_is_seen(case):
    Q, K, V, table, dO, kw, offset, p = inputs(case, "cpu")
    M, N, D, nb = Q.shape[2], K.shape[2], Q.shape[3], table.shape[0]
    keep = None
    if p:
        keep = torch.rand(*Q.shape[:3], N, generator=torch.Generator().manual_seed(1)) >= p
    want, bound = expected(Q, K, V, table, dO, offset=offset, keep=keep, p_drop=p, **kw)
    cols = 32 if D <= 64 else 64
    far = far_parts(M, N, nb, kw["max_distance"], kw["bidirectional"], offset, cols)
    near_only, _ = expected(Q, K, V, table, dO, offset=offset, keep=keep, p_drop=p, drop_pairs=far, **kw)
    missing = want - near_only  # doubled, they add as much; with the wrong sign twice that
    assert missing.norm() > 3 * bound.norm(), (missing.norm(dim=0) / bound.norm(dim=0)).tolist()
