"""The sampler where its sums decide at their limits. Tolerances as in test_sampling_gpu.py."""
import math
from decimal import Decimal, localcontext

import pytest
import torch

from tests.sampling_reference import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from starter_b200 import ops as ops_mod
    return ops_mod


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(64, 262144), (34, 524288), (130, 131072)])
@pytest.mark.parametrize("before", [0, 1])
def test_long_rows_of_equal_values(ops, dtype, rows, vocab, before):
    """All logits but one are equal, and a piece of 15 bits of their weight is nearly 2^15: 32715 and 32740, so that
    131284 and 131184 of them pass 2^32. Top-p cuts through the equal ones."""
    x = torch.full((rows, vocab + before), -0.419921875, dtype=dtype, device="cuda")[:, before:]
    x[1::2] = -0.42578125
    x[:, vocab - 5] = 0
    u = (torch.arange(rows) + 0.53) / rows
    tokens, logprobs = ops.sample_tokens(x, u.cuda(), top_p=0.9)
    for r in (0, 1, rows // 2, rows - 1):
        token, logprob, border = sample(x[r].cpu(), u[r].item(), top_p=0.9)
        assert border > 1e-7 and tokens[r].item() == token, r
        assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-7


# (x, z, u): with w = exp(x) and s = exp(z), w exceeds u (w + 1 + s) by 0.7 to 0.9 times 2^-44. x lies where the
# exponential's polynomial is worst: the Taylor series cut at the same degree is 1.3 to 2.4 units low there.
NEAR_A_BORDER = [
    (-0.5846397280693054, -18.968706130981445, 0.35786569118499756),
    (-0.3688790500164032, -16.71488380432129, 0.40881189703941345),
    (-0.1521206945180893, -17.41411590576172, 0.46204298734664917),
    (-0.02162468247115612, -18.41573715209961, 0.4945940375328064),
    (-0.4111839234828949, -17.23466682434082, 0.39862826466560364),
    (-0.3676796555519104, -18.10429573059082, 0.40910181403160095),
    (-0.28144463896751404, -18.25374984741211, 0.43009963631629944),
    (-0.02200602926313877, -16.6431884765625, 0.49449869990348816),
    (-0.4543777406215668, -17.165634155273438, 0.3883204162120819),
    (-0.19444704055786133, -19.032230377197266, 0.45154082775115967),
    (-0.3245144784450531, -19.37396240234375, 0.41957592964172363),
    (-0.021425563842058182, -17.46117401123047, 0.49464380741119385),
    (-0.06464847177267075, -18.126218795776367, 0.48384350538253784),
    (-0.49883729219436646, -16.706703186035156, 0.3778139352798462),
    (-0.15167127549648285, -16.506135940551758, 0.46215468645095825),
    (-0.10817883163690567, -17.925403594970703, 0.47298163175582886),
]


def test_weights_are_exact_to_less_than_a_unit(ops):
    """Token 0 is drawn if the weight of the first logit is not below 2^44 u (w + 1 + s). Two weights, each off by less than
    0.6 units, the first counting (1 - u) times and the other u times, are together off by less than 0.6."""
    x = torch.tensor([[a, 0.0, b] for a, b, _ in NEAR_A_BORDER])
    u = torch.tensor([u for _, _, u in NEAR_A_BORDER])
    with localcontext() as c:
        c.prec = 40
        for (a, b, _), e in zip(NEAR_A_BORDER, u.tolist()):
            w, s = Decimal(a).exp(), Decimal(b).exp()
            assert Decimal("0.7") < (w - Decimal(e) * (w + 1 + s)) * 2 ** 44 < Decimal("0.9")
    tokens, _ = ops.sample_tokens(x.cuda(), u.cuda())
    assert tokens.tolist() == [0] * len(u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1e36, 2e37, 3e38, math.inf])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=40), dict(top_k=700), dict(top_k=3000), dict(top_p=0.5), dict(min_p=0.2),
                                      dict(top_k=2500, top_p=0.7)], ids=str)
def test_logits_whose_differences_leave_32_bits(ops, dtype, temperature, settings):
    """From the type's lowest number nearly to its largest, at temperatures at which all of that weighs."""
    g = torch.Generator().manual_seed(44)
    x = ((torch.rand((5, 6001), generator=g) * 2 - 1) * 3.3e38).to(dtype)
    x[1, ::3] = torch.finfo(dtype).min
    x[2, 5] = torch.finfo(dtype).max
    x[3] = torch.where(torch.rand(6001, generator=g) < 0.5, -3.2e38, 3e38).to(dtype)
    x[4, 77] = math.inf
    u = torch.tensor([0.1234567, 0.4703, 0.987654, 0.7712, 0.3])
    tokens, logprobs = ops.sample_tokens(x.cuda(), u.cuda(), temperature=temperature, **settings)
    for r in range(4):
        token, logprob, border = sample(x[r], u[r].item(), temperature=temperature, **settings)
        assert border > 1e-7 and tokens[r].item() == token, (r, border)
        assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-7
    assert tokens[4].item() == 77 and logprobs[4].item() == 0
