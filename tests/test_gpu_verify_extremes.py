"""Verification where logits, temperatures or rows leave the ordinary range,
against the rule in 64 bits (test_gpu_verify.py, with its tolerances)."""
import math

import pytest
import torch

from test_gpu_verify import check, kvr, make  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temp", [0.3, 1.0])
@pytest.mark.parametrize("K", [0, 2])
def test_rows_of_the_types_lowest_value(kvr, dtype, temp, K):  # noqa: F811
    """A row masked throughout with the lowest value is a row of equal logits:
    drawn from evenly, after a full acceptance and where nothing is left."""
    V = 5003
    t, d, tokens, u, noise = make(8, K, V, dtype, temp, seed=11)
    low = torch.finfo(dtype).min
    t[:4, K] = low
    t[4:6, K, 100:] = low
    r = kvr.verify_draft_tokens(t, t[:, :K].contiguous(), tokens, u, noise, temperature=temp)
    assert (r.accepted == K).all()
    assert torch.equal(r.tokens[:4, K], noise[:4].argmin(-1)) and (r.tokens[4:6, K] < 100).all()
    check(kvr, (t, t[:, :K].contiguous(), tokens, u, noise), temp)
    if K:
        t[:, 0] = low                               # equal rows, refused: nothing is left of p - q
        r = kvr.verify_draft_tokens(t, t[:, :K].contiguous(), tokens, torch.ones_like(u), noise, temperature=temp)
        assert (r.accepted == 0).all() and torch.equal(r.tokens[:, 0], noise.argmin(-1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temp", [0.05, 1e-3, 1e-6, 1e-20, 2e-38])
@pytest.mark.parametrize("V", [37, 20011])
def test_small_temperatures(kvr, dtype, temp, V):  # noqa: F811
    """Only the largest logits have weight, and among equal ones the noise
    decides, however small the temperature."""
    t, _, _, u, noise = make(12, 3, V, dtype, 1.0, seed=V)
    t = t.round()                                   # many equal logits
    t[::2] += 1000                                  # (less than 2^11: exact in every type, up to a multiple of 4 or 8)
    t = t.contiguous()
    top = t[:, :3] == t[:, :3].amax(-1, keepdim=True)
    tokens = torch.where(top, torch.rand(top.shape, device="cuda"), -1.0).argmax(-1)
    check(kvr, (t, t[:, :3].contiguous(), tokens, u, noise), temp)
    r = kvr.verify_draft_tokens(t, t[:, :3].contiguous(), tokens, u, noise, temperature=temp)
    assert (r.accepted == 3).all()
    best = t[:, 3] == t[:, 3].amax(-1, keepdim=True)
    if temp <= 1e-3:
        assert torch.equal(r.tokens[:, 3], torch.where(best, noise, math.inf).argmin(-1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [100, 9001])
def test_equal_models_leave_nothing_to_draw_from(kvr, dtype, V):  # noqa: F811
    """Where p and q are equal their difference is 0, not a rounding error: a
    refusal (u = 1, a token outside the vocabulary) draws from p."""
    t, _, tokens, u, noise = make(60, 2, V, dtype, 0.8, seed=V)
    tokens[::2, 0] = V
    r = kvr.verify_draft_tokens(t, t[:, :2].contiguous(), tokens, torch.ones_like(u), noise, temperature=0.8)
    assert (r.accepted == 0).all()
    score = torch.softmax(t[:, 0].double() / 0.8, -1) / noise.double()
    top = score.topk(2).values
    sure = top[:, 1] < top[:, 0] * (1 - 2.0 ** -16)
    assert sure.double().mean() > 0.9 and torch.equal(r.tokens[sure, 0], score.argmax(-1)[sure])
