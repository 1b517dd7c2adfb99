"""Beam search's selection where more of a row reaches a part's threshold than there is room for, and at the ends of the logits' ranges."""
import math

import pytest
import torch

import kvmix_b200 as kv
from test_beam_reach_host import COINCIDING, coinciding

pytestmark = pytest.mark.gpu


def best(x, n):
    """Tokens of every row's n largest logits, equal ones by token."""
    return x.float().sort(dim=1, descending=True, stable=True).indices[:, :n].int()


# ---- more that reaches a part's threshold than there is room for -------------------------------------------------------------------------

@pytest.mark.parametrize("n,of", COINCIDING)
def test_a_token_with_the_number_of_the_thresholds_piece(cuda, n, of):
    """300 rows are one part each."""
    x = torch.randn(300, 131072, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda") - 12.0
    for row in (0, 150, 299):
        x[row] = torch.from_numpy(coinciding(n, of, 131072)[0]).cuda()
    for kind in ((torch.float16, torch.bfloat16) if of == 8 else (torch.float32,)):
        y = x.to(kind)
        assert torch.equal(kv.beam_select(y, torch.zeros(300, device="cuda"), 1, n=n).tokens, best(y, n))


@pytest.mark.parametrize("rows,V", [(1, 1 << 20), (150, 262144), (300, 131072), (297, 40000)])
@pytest.mark.parametrize("kind", [torch.float16, torch.float32])
def test_few_values_in_few_threads(cuda, rows, V, kind):
    """Thousands of equal numbers in the pieces of some threads that begin late in the row, single ones far apart: parts from one to 32."""
    gen = torch.Generator(device="cuda").manual_seed(V + rows)
    token = torch.arange(V, device="cuda")
    thread = token // (16 // (2 if kind is torch.float16 else 4)) % 256
    pick = lambda hi, size=(1,): torch.randint(hi, size, generator=gen, device="cuda")         # noqa: E731
    for n in (1, 2, 16, 17, 32, 33, 128):
        x = torch.full((rows, V), -10.0, device="cuda")
        dense = (thread < 8 + pick(60, (rows, 1))) & (token >= pick(V // 2, (rows, 1)))
        x[dense] = pick(3, (int(dense.sum()),)).float()
        x.scatter_(1, pick(V, (rows, 50)), 2.0)
        y = x.to(kind)
        assert torch.equal(kv.beam_select(y, torch.zeros(rows, device="cuda"), 1, n=n).tokens, best(y, n))
