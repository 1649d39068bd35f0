"""Operators of a serving step where they can go wrong: small vocabularies with many alternatives.  References and bounds are those of
test_serving_ops_gpu."""
import pytest
import torch

from test_serving_ops_gpu import TYPES, _check_logprobs, _gen, _randn, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# ── log probabilities ──────────────────────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [33, 40, 64, 100, 200, 255, 256, 258, 300, 511, 512, 513, 600])
def test_token_logprobs_small_vocabularies_with_many_alternatives(ops, dtype, vocab):
    """Rows with fewer 16-byte pieces than two warps, which start at every offset from a 16-byte boundary."""
    x = (_randn(_gen(vocab), 5, vocab + 3) * 3).to(dtype)
    for offset in range(4):
        for top_n in (31, 32, 33, 40, 64):
            if top_n <= vocab:
                _check_logprobs(ops, x[:, offset:offset + vocab], [0, vocab - 1, vocab // 2, -1, 7], top_n)


def test_token_logprobs_small_masked_vocabularies(ops):
    """The same where a mask leaves fewer tokens than alternatives are asked for."""
    x = torch.full((4, 100), -float("inf"), device="cuda")
    x[0, [5, 17, 99]] = torch.tensor([1.0, 3.0, 2.0], device="cuda")
    x[2, :] = 1.5
    x[3, :50] = float("nan")
    x[3, 50:] = _randn(_gen(1), 50)
    _check_logprobs(ops, x, [17, 0, 3, 70], 64)
