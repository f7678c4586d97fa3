"""Log-probabilities of given tokens with entropies and alternatives: the plain statement against the definition and against differences, and what it refuses."""
import math

import pytest
import torch

from torchtune_b200 import ops

INF = float("inf")


def _logits(*shape, seed=0, dtype=torch.float64):
    return (3 * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)).to(dtype)


@pytest.mark.parametrize("temperature", [1.0, 0.4])
@pytest.mark.parametrize("top", [0, 1, 5, 11])
def test_statement_against_the_definition(top, temperature):
    logits, tokens = _logits(2, 3, 11), torch.tensor([[0, 10, 4], [3, 3, 9]])
    s = ops.token_statistics(logits, tokens, temperature=temperature, top=top)
    assert (s.top_logprobs is None) == (s.top_tokens is None) == (top == 0)
    for at in ((0, 0), (1, 2), (0, 1)):
        z = [float(v) / temperature for v in logits[at]]
        total = sum(math.exp(v) for v in z)
        p = [math.exp(v) / total for v in z]
        assert math.isclose(float(s.logprobs[at]), math.log(p[int(tokens[at])]), rel_tol=1e-12)
        assert math.isclose(float(s.entropy[at]), -sum(q * math.log(q) for q in p), rel_tol=1e-12)
        best = sorted(range(11), key=lambda v: (-z[v], v))[:top]
        if top:
            assert s.top_tokens[at].tolist() == best
            torch.testing.assert_close(s.top_logprobs[at], torch.tensor([math.log(p[v]) for v in best], dtype=torch.float64), rtol=1e-12, atol=0)


def test_gradients_against_differences():
    logits, tokens = _logits(4, 7, seed=1), torch.tensor([0, 6, -100, 3])
    for top in (0, 3):
        assert torch.autograd.gradcheck(lambda x: tuple(t for t in ops.token_statistics(x, tokens, temperature=0.7, top=top)[:3] if t is not None), logits.requires_grad_())


def test_of_equal_logits_the_first_count():
    logits = torch.tensor([[1.0, 2.0, 2.0, 0.0, 2.0, -0.0, 1.0]])
    assert ops.token_statistics(logits, torch.tensor([0]), top=7).top_tokens.tolist() == [[1, 2, 4, 0, 6, 3, 5]]


def test_masked_logits():
    tokens = torch.tensor([0, 2, 0, 0, 1])
    logits = torch.tensor([[0.0, 0.0, -INF, -INF], [0.0, 0.0, -INF, -INF], [-INF] * 4, [0.0, float("nan"), 1.0, 2.0], [torch.finfo(torch.float32).min] * 4], requires_grad=True)
    s = ops.token_statistics(logits, tokens, top=3)
    (g,) = torch.autograd.grad(s.entropy[0] + s.logprobs[0], logits)
    s = s._replace(logprobs=s.logprobs.detach(), entropy=s.entropy.detach())
    assert math.isclose(float(s.logprobs[0]), -math.log(2), rel_tol=1e-6) and float(s.logprobs[1]) == -INF
    assert math.isclose(float(s.entropy[0]), math.log(2), rel_tol=1e-6) and s.entropy[2:4].isnan().all() and s.logprobs[2:4].isnan().all()
    assert math.isclose(float(s.logprobs[4]), -math.log(4), rel_tol=1e-6) and math.isclose(float(s.entropy[4]), math.log(4), rel_tol=1e-6)
    assert s.top_tokens.tolist() == [[0, 1, 2], [0, 1, 2], [0, 1, 2], [1, 3, 2], [0, 1, 2]]
    assert g[0].isfinite().all() and not g[0, 2:].any()


def test_ignored_tokens_keep_their_rows_entropy():
    logits = _logits(3, 9)
    some = ops.token_statistics(logits, torch.tensor([1, 5, 2]), top=2)
    s = ops.token_statistics(logits, torch.tensor([1, 7, 2]), top=2, ignore_index=7)
    assert float(s.logprobs[1]) == 0 and torch.equal(s.entropy, some.entropy) and torch.equal(s.top_tokens, some.top_tokens) and torch.equal(s.logprobs[[0, 2]], some.logprobs[[0, 2]])


def test_refusals():
    logits, tokens = _logits(3, 9), torch.tensor([1, 2, 3])
    for args, how in (((logits, tokens[:2]), {}), ((logits, tokens.int()), {}), ((logits.long(), tokens), {}), ((logits, tokens), dict(top=10)), ((logits, tokens), dict(top=-1)),
                      ((_logits(3, 99), tokens), dict(top=65)), ((logits, tokens), dict(temperature=0.0)), ((logits, tokens), dict(temperature=-1.0)), ((logits, tokens), dict(temperature=INF)),
                      ((logits, tokens), dict(temperature=float("nan"))), ((logits, torch.tensor([1, 2, 9])), {}), ((logits, torch.tensor([1, 2, -1])), {}), ((logits[:, :0], tokens), {}),
                      ((torch.tensor(1.0), torch.tensor(0)), {})):
        with pytest.raises(ValueError):
            ops.token_statistics(*args, **how)


def test_shapes_and_types():
    for shape in ((9,), (0, 9), (2, 0, 9), (2, 3, 2, 9)):
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            s = ops.token_statistics(_logits(*shape, dtype=dtype), torch.zeros(shape[:-1], dtype=torch.int64), top=2)
            assert s.logprobs.shape == s.entropy.shape == shape[:-1] and s.top_tokens.shape == s.top_logprobs.shape == (*shape[:-1], 2)
            assert s.logprobs.dtype == s.entropy.dtype == s.top_logprobs.dtype == torch.float32 and s.top_tokens.dtype == torch.int64
