"""Token log probabilities on the CPU: definition, gradient, refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import cuda_force_amd as cf
from cuda_force_amd import _lib, ops
from tests.logprobs_util import close, entropy_tolerance, gradient, logprob_tolerance, reference


@pytest.mark.parametrize("through", ["ops", "plain"])
@pytest.mark.parametrize("rows,vocab,count,top", [(1, 1, 1, 1), (4, 7, 3, 7), (5, 1001, 1, 20)])
def test_definition(through, rows, vocab, count, top):
    logits = 3 * torch.randn(rows, vocab)
    tokens = torch.randint(0, vocab, (rows, count))
    if through == "ops":
        got = cf.token_logprobs(logits, tokens, scale=0.7, entropy=True, top=top)
    else:
        got = ops._token_logprobs_reference(logits, tokens, 0.7, True, top)
    ref = reference(logits, tokens, 0.7, top)
    close(got[0], ref[0], logprob_tolerance(ref[0], vocab))
    close(got[1], ref[1], entropy_tolerance(ref[1], vocab))
    close(got[2], ref[2], logprob_tolerance(ref[2], vocab))
    assert torch.equal(got[3], ref[3])


def test_shapes_and_what_is_not_asked_for():
    logits = torch.randn(2, 3, 11)
    one = cf.token_logprobs(logits, torch.zeros(2, 3, dtype=torch.int32))
    assert one.logprobs.shape == (2, 3) and one.logprobs.dtype == torch.float32
    assert one.entropy is None and one.top_logprobs is None and one.top_tokens is None
    several = cf.token_logprobs(logits, torch.zeros(2, 3, 4, dtype=torch.int64), entropy=True, top=5)
    assert several.logprobs.shape == (2, 3, 4) and several.entropy.shape == (2, 3)
    assert several.top_logprobs.shape == several.top_tokens.shape == (2, 3, 5)
    row = cf.token_logprobs(logits[0, 0], torch.tensor(3), entropy=True, top=2)
    assert row.logprobs.shape == () and row.entropy.shape == () and row.top_tokens.shape == (2,)
    none = cf.token_logprobs(torch.empty(0, 5), torch.empty(0, dtype=torch.int64), entropy=True, top=2)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 2)


def test_padding_and_tokens_outside():
    got = cf.token_logprobs(torch.zeros(3, 4), torch.tensor([-100, 4, 1])).logprobs
    assert got[0] == 0 and got[1].isnan() and abs(got[2] + torch.tensor(4.0).log()) < 1e-6


def test_ties_masks_and_nan():
    inf = float("inf")
    logits = torch.tensor([[1.0, 2.0, 2.0, -0.0, 0.0], [-inf, 1.0, -inf, -inf, 1.0], [-inf] * 5,
                           [0.0, float("nan"), 1.0, 2.0, 3.0]])
    got = cf.token_logprobs(logits, torch.zeros(4, dtype=torch.int64), entropy=True, top=5)
    assert got.top_tokens.tolist() == [[1, 2, 0, 3, 4], [1, 4, 0, 2, 3], [0, 1, 2, 3, 4], [1, 4, 3, 2, 0]]
    assert abs(got.entropy[1] - torch.tensor(2.0).log()) < 1e-6
    assert got.logprobs[1] == -inf and got.logprobs[2].isnan() and got.logprobs[3].isnan()
    assert got.entropy[2].isnan() and got.entropy[3].isnan()


@pytest.mark.parametrize("with_g,with_h", [(True, False), (False, True), (True, True)])
def test_gradient_operator_is_the_formula_and_autograd(with_g, with_h):
    logits = torch.randn(6, 50)
    tokens = torch.randint(0, 50, (6, 3))
    tokens[0, 1] = tokens[0, 0]
    tokens[1] = -100
    tokens[2, 2] = -1
    g = torch.randn(6, 3) if with_g else None
    h = torch.randn(6) if with_h else None
    _, stats, entropy, _, _ = torch.ops.cudaforge.token_logprobs(logits, tokens, 0.8, True, 0)
    got = torch.ops.cudaforge.token_logprobs_backward(logits, tokens, 0.8, stats, entropy, g, h)
    ref, size = gradient(logits, tokens, 0.8, g, h)
    close(got, ref, 2.0**-20 * (size + 1e-6))
    leaf = logits.clone().requires_grad_(True)
    out = cf.token_logprobs(leaf, tokens, 0.8, entropy=True)
    outputs = ([out.logprobs] if with_g else []) + ([out.entropy] if with_h else [])
    auto, = torch.autograd.grad(outputs, [leaf], [v for v in (g, h) if v is not None])
    close(auto, ref, 2.0**-20 * (size + 1e-6))


def test_gradient_against_differences():
    logits = torch.randn(3, 9, dtype=torch.float64, requires_grad=True)
    tokens = torch.tensor([[1, 1], [-1, 4], [0, 8]])

    def f(x):
        got = cf.token_logprobs(x, tokens, 1.3, entropy=True)
        return got.logprobs, got.entropy

    assert torch.autograd.gradcheck(f, (logits,))


def test_refusals():
    logits, tokens = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, 1, 1, dtype=torch.int64),
                torch.zeros(2, 3, dtype=torch.int64), torch.zeros(3, 0, dtype=torch.int64),
                torch.zeros(3, 1025, dtype=torch.int64)):
        with pytest.raises(ValueError):
            cf.token_logprobs(logits, bad)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            cf.token_logprobs(logits, tokens, scale)
    for top in (-1, 6):
        with pytest.raises(ValueError):
            cf.token_logprobs(logits, tokens, top=top)
    with pytest.raises(ValueError):
        cf.token_logprobs(torch.zeros(3, 100), tokens, top=65)
    with pytest.raises(TypeError):
        cf.token_logprobs(logits, tokens.float())
    with pytest.raises(ValueError):
        cf.token_logprobs(torch.zeros(3, 0), tokens)


def test_c_abi_refusals_before_any_launch():
    lib = _lib.load()
    fake = ctypes.c_void_p(0x1000)
    null = ctypes.c_void_p(0)

    def forward(dtype=0, rows=4, vocab=100, stride=100, tokens=fake, count=1, scale=1.0, out=fake, top=0, top_out=fake,
                ws=fake, ws_bytes=1 << 30, logits=fake):
        return lib.cf_token_logprobs(logits, dtype, rows, vocab, stride, tokens, count, scale, out, null, null, top,
                                     top_out, top_out, ws, ws_bytes, null)

    assert forward(rows=0) == _lib.CF_OK and forward(vocab=0) == _lib.CF_OK
    bad = _lib.CF_ERR_INVALID_ARGUMENT
    for case in ({"dtype": 7}, {"stride": 99}, {"tokens": null}, {"logits": null}, {"count": 0}, {"count": 1025},
                 {"scale": 0.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"out": null}, {"top": -1},
                 {"top": 65}, {"top": 101}, {"top": 3, "top_out": null}, {"vocab": 2**27 + 1, "stride": 2**28},
                 {"rows": 2**31}, {"logits": ctypes.c_void_p(0x1002)},
                 {"vocab": 50000, "stride": 50000, "ws_bytes": 0}, {"vocab": 50000, "stride": 50000, "ws": null}):
        assert forward(**case) == bad, case
    assert lib.cf_token_logprobs_workspace_bytes(0, 100000, 1000, 5) == 0
    assert lib.cf_token_logprobs_workspace_bytes(2, 1, 50257, 20) > 0

    def backward(stats=fake, entropy=fake, h=null, grad=fake, stride=100):
        return lib.cf_token_logprobs_backward(fake, 0, 4, 100, 100, fake, 1, 1.0, stats, entropy, fake, h, grad,
                                              stride, null)

    for case in ({"stats": null}, {"grad": null}, {"entropy": null, "h": fake}, {"stride": 99},
                 {"grad": ctypes.c_void_p(0x1001)}):
        assert backward(**case) == bad, case


def test_the_entropys_gradient_does_not_ask_for_the_tokens():
    logits = torch.randn(3, 30)
    tokens = torch.tensor([[5], [30], [-1]])
    h = torch.randn(3)
    _, stats, entropy, _, _ = torch.ops.cudaforge.token_logprobs(logits, tokens, 0.8, True, 0)
    got = torch.ops.cudaforge.token_logprobs_backward(logits, tokens, 0.8, stats, entropy, None, h)
    ref, size = gradient(logits, tokens.clamp(max=0), 0.8, None, h)
    close(got, ref, 2.0**-20 * (size + 1e-6))


@pytest.mark.parametrize("through", ["ops", "kernels"])
def test_a_row_of_padding_alone_has_no_gradient_whatever_it_holds(through):
    logits = torch.randn(4, 6)
    logits[1] = float("-inf")
    logits[2, 3] = float("nan")
    tokens = torch.tensor([[1, 2], [-1, -100], [-1, -1], [-1, 5]])
    g, h = torch.ones(4, 2), torch.tensor([0.5, 0.0, 0.0, 0.0])
    for with_h in (False, True):
        if through == "ops":
            leaf = logits.clone().requires_grad_()
            got = cf.token_logprobs(leaf, tokens, 0.9, entropy=True)
            grad, = torch.autograd.grad(got.logprobs, leaf, g)
        else:
            _, stats, entropy, _, _ = torch.ops.cudaforge.token_logprobs(logits, tokens, 0.9, True, 0)
            grad = torch.ops.cudaforge.token_logprobs_backward(logits, tokens, 0.9, stats, entropy, g,
                                                               h if with_h else None)
        assert (grad[1:3] == 0).all() and torch.isfinite(grad).all() and (grad[[0, 3]] != 0).all()
    if through == "kernels":
        alone = torch.ops.cudaforge.token_logprobs_backward(logits, tokens, 0.9, stats, entropy, None, h)
        assert (alone[1:] == 0).all() and (alone[0] != 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_logits_at_the_ends_of_their_type_keep_their_differences_when_scaled(dtype):
    low = torch.finfo(dtype).min
    logits = torch.full((2, 8), low, dtype=dtype)
    logits[1, 3] = 1.0
    tokens = torch.tensor([2, 3])
    leaf = logits.clone().requires_grad_()
    for got in (cf.token_logprobs(logits, tokens, 2.0, entropy=True, top=2),
                cf.token_logprobs(leaf, tokens, 2.0, entropy=True, top=2)):
        assert abs(got.logprobs[0] + torch.tensor(8.0).log()) < 1e-6 and got.logprobs[1] == 0
        assert abs(got.entropy[0] - torch.tensor(8.0).log()) < 1e-6 and got.entropy[1] == 0
        assert got.top_tokens.tolist() == [[0, 1], [3, 0]]
    got.logprobs.sum().backward()
    want = torch.full((8,), -0.25)
    want[2] += 2.0
    assert (leaf.grad[0].float() - want).abs().max() < 1e-6 and (leaf.grad[1] == 0).all()
