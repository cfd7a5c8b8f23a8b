"""The sampler where its sums decide at their limits. Tolerances as in test_sampling_gpu.py."""
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
def test_long_rows_of_equal_values(ops, dtype, rows, vocab):
    """All logits but one are equal, and a piece of 15 bits of their weight is nearly 2^15: 32715 and 32740, so that
    131284 and 131184 of them pass 2^32. Top-p cuts through the equal ones."""
    x = torch.full((rows, vocab), -0.419921875, dtype=dtype, device="cuda")
    x[1::2] = -0.42578125
    x[:, vocab - 5] = 0
    u = (torch.arange(rows) + 0.53) / rows
    tokens, logprobs = ops.sample_tokens(x, u.cuda(), top_p=0.9)
    for r in (0, 1, rows // 2, rows - 1):
        token, logprob, border = sample(x[r].cpu(), u[r].item(), top_p=0.9)
        assert border > 1e-7 and tokens[r].item() == token, r
        assert abs(logprobs[r].item() - logprob) <= 2.0 ** -24 * abs(logprob) + 1e-7
