"""The 64-bit restatements in oracle/token_ops_oracle.py against hand-worked values and differences (CPU)."""
import math

import torch

from oracle import token_ops_oracle as O


def test_top_logits_order_and_tail():
    x = torch.tensor([[1.0, 3.0, -0.0, 3.0, 0.0, math.nan, -math.inf]])
    v, i, t = O.top_logits(x, 4)
    assert i.tolist() == [[5, 1, 3, 0]] and math.isnan(v[0, 0])
    assert abs(t.item() - math.log(2)) < 1e-12                 # the two zeros and exp(-inf)
    assert O.top_logits(x[:, :3], 3)[2].item() == -math.inf


def test_gradients_by_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((3, 4, 9), generator=g, dtype=torch.float64).requires_grad_(True)
    y = torch.randint(1, 9, (3, 4), generator=g)
    y[2, 1] = 0
    v, i, t = O.top_logits(torch.randn((3, 4, 9), generator=g), 3, 1.5)
    old, ref = -2 + 0.1 * torch.randn((3, 4), generator=g), -2 + 0.1 * torch.randn((3, 4), generator=g)
    adv = torch.randn((4,), generator=g)
    seq = -8 + torch.randn((4,), generator=g)
    check = lambda f: torch.autograd.gradcheck(f, (x,))  # noqa: E731
    assert check(lambda z: O.token_logprob(z, y, 0, 0.7))
    assert check(lambda z: O.distill_rows(z, v, i, y, 0, t, 1.5, 0.3))
    assert check(lambda z: O.policy_rows(z, y, 0, old, adv, ref, 0.2, 0.3, 0.1, 0.05)[0])
    assert check(lambda z: O.preference(z, y, 0, seq, 0.3, 0.1)[0])


def test_distillation_of_the_own_distribution_is_zero_and_of_a_point_is_cross_entropy():
    x = torch.randn(1, 2, 11, dtype=torch.float64)
    y = torch.ones(1, 2, dtype=torch.long)
    v, i, t = O.top_logits(x, 4, 2.0)
    assert O.distill_rows(x, v, i, y, 0, t, 2.0).abs().max() < 1e-12
    one = torch.zeros(1, 2, 1)
    ce = -torch.log_softmax(x, -1)[..., 5]
    assert torch.allclose(O.distill_rows(x, one, torch.full((1, 2, 1), 5), y, 0), ce)


def test_policy_and_preference_values():
    x = torch.zeros(1, 2, 4, dtype=torch.float64)
    y = torch.ones(1, 2, dtype=torch.long)
    lp = torch.full((1, 2), -math.log(4.0))
    rows, _, ent = O.policy_rows(x, y, 0, lp - 1, torch.tensor([1.0, -1.0]))
    assert torch.allclose(rows, torch.tensor([[-1.2, math.e]], dtype=torch.float64)) and torch.allclose(ent, -lp.double())
    loss, seq = O.preference(x, y, 0, torch.tensor([-math.log(4.0), 1.0 - math.log(4.0)]), beta=1.0)
    assert abs(loss.item() - math.log1p(math.exp(-1.0))) < 1e-7 and torch.allclose(seq, lp[0].double())
