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


# ---- logits far from zero -----------------------------------------------------------------------------------------------------------------

def log_softmax(x):
    """In 64 bits; the largest logit and the logarithm are not added up, which loses the latter beside a large one."""
    top = x.amax(1, keepdim=True)
    return (x - top) - (x - top).exp().sum(1, keepdim=True).log()


def definition(logits, scores, beams, n, ends):
    """As test_gpu_beams.definition, whose `x - logsumexp(x)` gives 0 in place of -log V where all logits are alike and large."""
    x = logits.double().cpu()
    value = scores.double().cpu()[:, None] + log_softmax(x)
    value[~(torch.isfinite(torch.logsumexp(x, 1)) & torch.isfinite(scores.cpu()))] = -math.inf
    out = []
    for r in range(x.shape[0] // beams):
        flat = value[r * beams:(r + 1) * beams].flatten()
        at = torch.sort(flat, descending=True, stable=True).indices[:n + 40].tolist()
        out.append([(float(flat[i]), i // x.shape[1], i % x.shape[1]) for i in at])
    return out


@pytest.fixture
def base(monkeypatch):
    import test_gpu_beams
    monkeypatch.setattr(test_gpu_beams, "definition", definition)
    return test_gpu_beams


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 100, 32000])
def test_rows_alike_anywhere(cuda, base, kind, V):
    """Every token of a row of equal logits has the probability 1 / V, whatever the logits."""
    huge, low = torch.finfo(kind).max, torch.finfo(kind).min
    x = torch.tensor([low, -30000.0, 0.0, huge] + ([] if kind is torch.float16 else [-1e30, 1e30, -1e9, 7e20]))[:, None].repeat(1, V).to(kind).cuda()
    scores = -torch.arange(float(len(x)), device="cuda")
    assert (log_softmax(x.double().cpu()) - torch.log_softmax(x.double().cpu(), 1)).abs().max() < 1e-12
    for beams in (1, 4):
        for n in {min(beams * V, n) for n in (beams, 2 * beams, 128)}:
            got = base.check(x, scores, beams, n)
            if beams == 1:
                assert (got.scores[:, 0] - (scores - math.log(V))).abs().max() <= 2.0 ** -18         # sums 2^-22, scores down to -18 rounded to 2^-20


@pytest.mark.parametrize("mask", [-3.0e38, -1e30, -1e10])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_a_masked_beam_does_not_pass_a_live_one(cuda, base, kind, mask):
    """A beam whose logits are all masked is worth its score less log V a token, less than a beam behind it that is sure of its next token."""
    x = torch.full((8, 32000), mask, device="cuda").to(kind)
    x[1::2] = base.inputs(4, 32000, kind, 5)[0]
    x[1::2, 77] = 40.0
    got = base.check(x, torch.tensor([-12.0, -15.0] * 4).cuda(), 2)
    assert (got.beams[:, 0] == 1).all() and (got.tokens[:, 0] == 77).all() and (got.beams[:, 1] == 0).all()
    assert (got.scores[:, 1] - (-12.0 - math.log(32000))).abs().max() <= 2.0 ** -18


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_large_logits_that_differ(cuda, base, kind):
    """Neighbouring numbers of the type at 2^100: the difference decides, not what is left of it beside the sum."""
    gen = torch.Generator().manual_seed(6)
    step = 2.0 ** (100 - (7 if kind is torch.bfloat16 else 23))
    x = torch.tensor([2.0 ** 100, -2.0 ** 101])[:, None] + step * torch.randint(0, 3, (2, 5000), generator=gen)
    x = x.to(kind).repeat(3, 1).cuda()
    base.check(x, -torch.rand(6, generator=gen).cuda(), 2, 64)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, torch.float32])
def test_masks_and_numbers_that_are_none(cuda, base, kind):
    base.test_masks_and_numbers_that_are_none(cuda, kind)
