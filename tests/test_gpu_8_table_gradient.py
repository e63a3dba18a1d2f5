"""The gradient of the table against 64 bits within the statistical bound of table_gradient_bound.py: batches, ragged
lengths, offsets, padding, holes, dropout and every width, at sizes where most of it comes from the far sums."""
import pytest
import torch

import fast_ops_b200._lib as L
from fast_ops_b200.flash_attention import dropout_mask, relative_attention
from table_gradient_bound import CASES, expected, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", CASES, ids=[c[0] for c in CASES])
def test_table_gradient_within_the_roundings_of_delta(case, cuda_device):
    Q, K, V, table, dO, kw, offset, p = inputs(case, "cuda")
    rng = (77, 4)
    keep = dropout_mask(p, *Q.shape[:3], K.shape[2], Q.device, rng=rng) if p else None
    t = table.clone().requires_grad_()
    O = relative_attention(Q, K, V, t, query_offset=offset, dropout_p=p, rng=rng if p else None, **kw)
    dT, = torch.autograd.grad(O, t, dO)
    want, bound = expected(Q, K, V, table, dO, offset=offset, keep=keep, p_drop=p, **kw)
    off = (dT.double() - want).norm(dim=0) / bound.norm(dim=0)
    assert off.max().item() <= 1.0, off.tolist()
    torch.cuda.synchronize()
    assert L.device_status(0) == 0
