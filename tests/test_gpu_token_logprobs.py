"""Token log probabilities on the GPU against float64."""

from __future__ import annotations

import pytest
import torch

import cuda_force_amd as cf
from tests.logprobs_util import close, entropy_tolerance, gradient, logprob_tolerance, reference

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(logits, tokens, scale=1.0, top=0):
    """All outputs; every repeat has the same bits."""
    got = cf.token_logprobs(logits, tokens, scale=scale, entropy=True, top=top)
    vocab = logits.shape[-1]
    given = tokens.reshape(logits.shape[0], -1)
    ref = reference(logits, given, scale, top)
    close(got.logprobs.reshape(given.shape), ref[0], logprob_tolerance(ref[0], vocab))
    close(got.entropy, ref[1], entropy_tolerance(ref[1], vocab))
    if top:
        close(got.top_logprobs, ref[2], logprob_tolerance(ref[2], vocab))
        assert torch.equal(got.top_tokens.cpu(), ref[3])
    again = cf.token_logprobs(logits, tokens, scale=scale, entropy=True, top=top)
    for a, b in zip(got, again):
        assert a is None and b is None or torch.equal(a.view(torch.int32), b.view(torch.int32))
    bare = cf.token_logprobs(logits, tokens, scale=scale).logprobs
    close(bare.reshape(given.shape), ref[0], logprob_tolerance(ref[0], vocab))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 64), (4, 255, 5), (1, 2049, 20), (9, 4100, 1), (300, 513, 8),
    (2, 32001, 64), (17, 50257, 20), (1200, 1001, 3), (1100, 33000, 5), (1, 300007, 33),
])
def test_sizes(dtype, rows, vocab, top):
    logits = (3 * torch.randn(rows, vocab, device="cuda")).to(dtype)
    check(logits, torch.randint(0, vocab, (rows,), device="cuda"), 1.25, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_padded_and_misaligned_rows(dtype, offset):
    wide = torch.randn(6, 1300, device="cuda").to(dtype)
    wide[:, 1100:] = float("nan")
    wide[:, :offset] = float("nan")
    logits = wide[:, offset:1100]
    check(logits, torch.randint(0, 1000, (6, 4), device="cuda"), 0.9, 10)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(4, 3000), (1500, 600)])
def test_masks_and_the_ends_of_the_range(dtype, rows, vocab):
    info = torch.finfo(dtype)
    logits = torch.randn(rows, vocab, device="cuda").to(dtype)
    logits[0, :] = float("-inf")
    logits[0, vocab // 2] = 1.0  # one token left
    logits[1, 1:] = info.min     # masked by the lowest value
    logits[2, :] = info.min      # nothing above it: uniform
    logits[3, : vocab - 3] = float("-inf")
    check(logits, torch.full((rows,), vocab // 2, device="cuda"), 1.0, 7)
    logits[0] = info.max
    logits[1, 5] = info.max
    check(logits, torch.full((rows,), 5, device="cuda"), 1.0, 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(5, 3000), (1500, 600)])
def test_rows_that_give_nan(dtype, rows, vocab):
    logits = torch.randn(rows, vocab, device="cuda").to(dtype)
    logits[0] = float("-inf")
    logits[1, 77] = float("nan")
    logits[1, 5] = float("nan")
    logits[2, 99] = float("inf")
    logits[3] = float("nan")
    got = cf.token_logprobs(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), entropy=True, top=4)
    ref = reference(logits, torch.zeros(rows, 1, dtype=torch.int64), 1.0, 4)
    for row in range(4):
        assert got.logprobs[row].isnan() and got.entropy[row].isnan()
    assert torch.equal(got.top_tokens.cpu(), ref[3])
    close(got.logprobs[4:], ref[0][4:, 0], logprob_tolerance(ref[0][4:, 0], vocab))


@pytest.mark.parametrize("rows,vocab", [(2, 70000), (1100, 4000)])
def test_a_common_offset_costs_nothing(rows, vocab):
    logits = 2 * torch.randn(rows, vocab, device="cuda") + 5000.0
    check(logits, torch.randint(0, vocab, (rows,), device="cuda"), 1.3, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 1100])
def test_ties_go_to_the_lowest_token(dtype, rows):
    vocab = 9000
    logits = torch.zeros(rows, vocab, device="cuda", dtype=dtype)
    logits[0, 4000:] = -0.0
    check(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), 1.0, 64)
    logits += torch.randint(0, 3, (rows, vocab), device="cuda").to(dtype)
    check(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), 1.0, 64)
    ordered = torch.arange(vocab, device="cuda").float().mul(-0.01).to(dtype).expand(rows, vocab).contiguous()
    check(ordered, torch.zeros(rows, dtype=torch.int64, device="cuda"), 1.0, 40)
    check(ordered.flip(1).contiguous(), torch.zeros(rows, dtype=torch.int64, device="cuda"), 1.0, 40)


def test_more_candidates_than_the_filter_holds():
    """A few threads of a workgroup own all the large logits (vectors are dealt
    to 256 threads in turn)."""
    rows, vocab = 1100, 131072
    logits = torch.zeros(rows, vocab, device="cuda", dtype=torch.bfloat16)
    vectors = logits.view(rows, -1, 256, 8)
    vectors[:, :, 3:5] = (1 + torch.rand(rows, vectors.shape[1], 2, 8, device="cuda")).to(torch.bfloat16)
    got = cf.token_logprobs(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=64)
    order = torch.sort(logits[:40], dim=-1, descending=True, stable=True).indices[:, :64]
    assert torch.equal(got.top_tokens[:40], order)


def test_more_keys_than_the_join_holds():
    """Every chunk of a split row (4096 logits here) brings nearly as many keys
    as are wanted, one chunk's second key below most of them."""
    vocab = 131072
    logits = torch.zeros(1, vocab, device="cuda", dtype=torch.bfloat16)
    chunks = logits.view(-1, 4096)
    chunks[1:, 100:163] = (101 + 20 * torch.rand(chunks.shape[0] - 1, 63, device="cuda")).to(torch.bfloat16)
    chunks[0, 50:52] = 100.0
    check(logits, torch.zeros(1, dtype=torch.int64, device="cuda"), 0.1, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,count", [(1, 5, 1), (7, 999, 3), (3, 32001, 1), (40, 50257, 1), (1200, 640, 2),
                                              (4, 3001, 300)])
@pytest.mark.parametrize("with_g,with_h", [(True, False), (False, True), (True, True)])
def test_gradient(dtype, rows, vocab, count, with_g, with_h):
    logits = (2 * torch.randn(rows, vocab, device="cuda")).to(dtype).requires_grad_(True)
    tokens = torch.randint(0, vocab, (rows, count), device="cuda")
    if count > 1:
        tokens[:, 1] = tokens[:, 0]
    tokens[rows // 2] = -100
    g = torch.randn(rows, count, device="cuda") if with_g else None
    h = torch.randn(rows, device="cuda") if with_h else None
    got = cf.token_logprobs(logits, tokens, 0.8, entropy=True, top=2)
    outputs = ([got.logprobs] if with_g else []) + ([got.entropy] if with_h else [])
    grad, = torch.autograd.grad(outputs, [logits], [v for v in (g, h) if v is not None], retain_graph=True)
    assert grad.dtype == dtype
    ref, size = gradient(logits, tokens, 0.8, g, h)
    # One rounding to the logits' type (half an ulp; the smallest subnormal for
    # what underflows), and fp32 errors of p and the entropy relative to the terms.
    tolerance = torch.finfo(dtype).eps / 2 * ref.abs() + (2.0**-18 + 8 * 2.0**-24 * vocab / 256) * size
    tolerance = tolerance + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    close(grad, ref, tolerance)
    again, = torch.autograd.grad(outputs, [logits], [v for v in (g, h) if v is not None])
    assert torch.equal(grad.view(torch.uint8), again.view(torch.uint8))


def test_gradient_of_padded_logits_and_padding_rows():
    wide = torch.randn(8, 1100, device="cuda", dtype=torch.bfloat16)
    logits = wide[:, 3:1007].requires_grad_(True)
    tokens = torch.tensor([5, -1, 7, 1003, -100, 0, 1, 2], device="cuda")
    g = torch.randn(8, device="cuda")
    got = cf.token_logprobs(logits, tokens)
    grad, = torch.autograd.grad(got.logprobs, logits, g)
    ref, size = gradient(logits, tokens[:, None], 1.0, g[:, None], None)
    close(grad, ref, 2.0**-8 * ref.abs() + 2.0**-18 * size)
    assert (grad[1] == 0).all() and (grad[4] == 0).all()
    loss = cf.token_logprobs(logits, tokens).logprobs.sum()
    loss.backward()  # accumulates into the view's own gradient
    assert logits.grad.shape == logits.shape


def test_a_token_outside_the_vocabulary_gives_nan_and_its_row_alone():
    logits = torch.randn(3, 50, device="cuda", requires_grad=True)
    got = cf.token_logprobs(logits, torch.tensor([1, 50, 2], device="cuda")).logprobs
    assert got[1].isnan() and not got[0].isnan() and not got[2].isnan()
    got.nansum().backward()
    assert not logits.grad[0].isnan().any() and not logits.grad[2].isnan().any()


def test_second_derivatives_are_refused():
    logits = torch.randn(3, 50, device="cuda", requires_grad=True)
    got = cf.token_logprobs(logits, torch.tensor([1, 2, 3], device="cuda")).logprobs
    grad, = torch.autograd.grad(got.sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_general_way_equals_direct():
    logits = torch.randn(4, 3, 700, device="cuda", dtype=torch.float16)
    tokens = torch.randint(0, 700, (4, 3), device="cuda", dtype=torch.int32)
    general = cf.token_logprobs(logits, tokens, 0.5, True, 6)
    direct = cf.token_logprobs(logits.view(12, 700), tokens.view(12).long(), 0.5, True, 6)
    for a, b in zip(general, direct):
        assert torch.equal(a.reshape(b.shape), b)
    columns = torch.randn(700, 12, device="cuda").t()  # not dense along the vocabulary: copied
    a = cf.token_logprobs(columns, tokens.view(12).long(), top=3)
    b = cf.token_logprobs(columns.contiguous(), tokens.view(12).long(), top=3)
    assert all(x is None or torch.equal(x, y) for x, y in zip(a, b))


def test_another_stream_and_a_replayed_graph():
    logits = torch.randn(8, 50257, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(0, 50257, (8,), device="cuda")
    eager = cf.token_logprobs(logits, tokens, entropy=True, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cf.token_logprobs(logits, tokens, entropy=True, top=20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cf.token_logprobs(logits, tokens, entropy=True, top=20)
        grad = torch.ops.cudaforge.token_logprobs_backward(
            logits, tokens[:, None], 1.0, *torch.ops.cudaforge.token_logprobs(logits, tokens[:, None], 1.0, True, 0)[1:3],
            torch.ones(8, 1, device="cuda"), None)
    for step in range(3):
        logits.copy_(torch.randn(8, 50257, device="cuda"))
        tokens.copy_(torch.randint(0, 50257, (8,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = cf.token_logprobs(logits, tokens, entropy=True, top=20)
        assert all(torch.equal(a, b) for a, b in zip(eager, out)), step
        leaf = logits.clone().requires_grad_(True)
        cf.token_logprobs(leaf, tokens, entropy=True).logprobs.sum().backward()
        assert torch.equal(leaf.grad, grad), step


def test_empty():
    got = cf.token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"),
                            entropy=True, top=3)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 3)


@pytest.mark.parametrize("shape", [(6,), (6, 3)], ids=["one", "several"])
@pytest.mark.parametrize("entropy, top", [(False, 0), (True, 0), (False, 4), (True, 4)])
def test_gradients_of_the_native_node_equal_the_general_ones(shape, entropy, top):
    # Three dimensions take the general way, two the native node: the same kernels.
    logits = torch.randn(6, 700, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(-1, 700, shape, device="cuda")
    two, three = logits.clone().requires_grad_(), logits.clone().view(1, 6, 700).requires_grad_()
    a = cf.token_logprobs(two, tokens, 0.7, entropy, top)
    b = cf.token_logprobs(three, tokens.view(1, *shape), 0.7, entropy, top)
    assert a.logprobs.requires_grad and a.logprobs.shape == shape and torch.equal(a.logprobs, b.logprobs[0])
    weights = torch.randn(shape, device="cuda")
    losses = [(r.logprobs.view(shape) * weights).sum() for r in (a, b)]
    if entropy:
        losses = [l + r.entropy.square().sum() for l, r in zip(losses, (a, b))]
    if top:
        assert not a.top_logprobs.requires_grad and not a.top_tokens.requires_grad
        assert torch.equal(a.top_tokens, b.top_tokens[0])
    for loss in losses:
        loss.backward()
    assert torch.equal(two.grad, three.grad[0])


def test_gradient_of_the_entropy_alone():
    logits = torch.randn(5, 333, device="cuda", requires_grad=True)
    got = cf.token_logprobs(logits, torch.zeros(5, dtype=torch.int64, device="cuda"), 1.0, True)
    got.entropy.sum().backward()
    x = logits.detach().cpu().double().requires_grad_()
    p = x.log_softmax(-1)
    (-(p.exp() * p).sum()).backward()
    # p (ln p + H) in fp32: a few roundings of values below 8, times p.
    assert (logits.grad.cpu().double() - x.grad).abs().max() <= 64 * 2.0 ** -24


def test_saved_tensors_are_guarded_and_may_be_packed():
    logits = torch.randn(4, 256, device="cuda", requires_grad=True)
    tokens = torch.tensor([1, 2, 3, 4], device="cuda")
    plain = cf.token_logprobs(logits, tokens).logprobs
    want, = torch.autograd.grad(plain.sum(), logits)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        packed = cf.token_logprobs(logits, tokens).logprobs
    got, = torch.autograd.grad(packed.sum(), logits)
    assert torch.equal(got, want)
    changed = cf.token_logprobs(logits, tokens).logprobs
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        changed.sum().backward()


@pytest.mark.parametrize("scale, top, count", [(float("nan"), 0, 1), (float("inf"), 0, 1), (1e29, 0, 1), (1.0, 65, 1),
                                               (1.0, 0, 1025)])
def test_limits_are_refused_alike_on_the_gpu(scale, top, count):
    with pytest.raises(ValueError):
        cf.token_logprobs(torch.zeros(2, 100, device="cuda"), torch.zeros(2, count, dtype=torch.int64, device="cuda"),
                          scale, top=top)


@pytest.mark.parametrize("padding, pitch", [(0, 500), (12, 512), (4500, 500)])
def test_the_gradient_takes_no_more_memory_than_the_logits(padding, pitch):
    # Rows behind a little padding keep their pitch; rows far apart (the last
    # position of every sequence) do not.
    whole = torch.randn(4, 500 + padding, device="cuda")
    logits = whole[:, :500].requires_grad_()
    tokens = torch.tensor([0, 1, 498, 499], device="cuda")
    got = cf.token_logprobs(logits, tokens).logprobs
    grad, = torch.autograd.grad(got.sum(), logits)
    ref, size = gradient(logits, tokens[:, None], 1.0, torch.ones(4, 1), None)
    close(grad, ref, 2.0**-24 * ref.abs() + (2.0**-18 + 8 * 2.0**-24 * 500 / 256) * size)
    direct = torch.ops.cudaforge.token_logprobs_backward(
        logits.detach(), tokens[:, None].contiguous(), 1.0,
        torch.ops.cudaforge.token_logprobs(logits.detach(), tokens[:, None].contiguous(), 1.0, False, 0)[1],
        torch.empty(0, device="cuda"), torch.ones(4, 1, device="cuda"), None)
    assert direct.stride() == (pitch, 1) and torch.equal(direct, grad)


def test_forward_and_backward_captured_and_replayed():
    """No eager graph of the same leaf lives while the capture runs."""
    logits = torch.randn(33, 1000, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(-1, 1000, (33,), device="cuda")
    weights = torch.randn(33, device="cuda")

    def step(leaf):
        got = cf.token_logprobs(leaf, tokens, 0.9, True)
        grad, = torch.autograd.grad([got.logprobs, got.entropy], [leaf], [weights, weights])
        return got.logprobs.detach(), got.entropy.detach(), grad

    static = logits.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static.detach().requires_grad_())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        results = step(static.detach().requires_grad_())
    for i in range(4):
        logits = torch.randn_like(logits)
        static.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(results, step(logits.clone().requires_grad_())):
            assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [1, 2, 3])
def test_as_many_chunks_as_a_row_can_have(rows):
    vocab = (1 << 22) + 3
    logits = torch.randn(rows, vocab, device="cuda", dtype=torch.bfloat16)
    check(logits, torch.full((rows,), vocab - 1, device="cuda"), 1.0, 64)


def test_rows_that_take_more_than_one_launch():
    """More rows than a launch has workgroups (2^24 of 256 threads)."""
    rows, vocab = 2**24 + 100, 8
    logits = torch.randn(rows, vocab, device="cuda", dtype=torch.bfloat16).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    got = cf.token_logprobs(logits, tokens, 0.7, True, 2)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    grad, = torch.autograd.grad([got.logprobs, got.entropy], [logits], [g, h])
    for at in (slice(0, 50), slice(2**24 - 50, rows)):
        ref = reference(logits[at], tokens[at, None], 0.7, 2)
        close(got.logprobs[at, None], ref[0], logprob_tolerance(ref[0], vocab))
        close(got.entropy[at], ref[1], entropy_tolerance(ref[1], vocab))
        close(got.top_logprobs[at], ref[2], logprob_tolerance(ref[2], vocab))
        assert torch.equal(got.top_tokens[at].cpu(), ref[3])
        want, size = gradient(logits[at], tokens[at, None], 0.7, g[at, None], h[at])
        close(grad[at], want, 2.0**-8 * want.abs() + 2.0**-18 * size + 2.0**-130)


def test_the_entropys_gradient_does_not_ask_for_the_tokens():
    """A token past the vocabulary gives a log probability of NaN, and its
    gradient too, but where only the entropy is differentiated no token counts."""
    for dtype in DTYPES:
        for count in (1, 3):
            logits = torch.randn(3, 300, device="cuda").to(dtype).requires_grad_()
            tokens = torch.tensor([[5], [300], [-1]], device="cuda").repeat(1, count)
            got = cf.token_logprobs(logits, tokens, 0.8, True)
            h = torch.randn(3, device="cuda")
            grad, = torch.autograd.grad(got.entropy, logits, h, retain_graph=True)
            ref, size = gradient(logits, tokens.clamp(max=0), 0.8, None, h)
            close(grad, ref, torch.finfo(dtype).eps / 2 * ref.abs() + 2.0**-18 * size + torch.finfo(dtype).tiny)
            both, = torch.autograd.grad([got.entropy, got.logprobs], logits, [h, torch.ones_like(got.logprobs)])
            assert both[1].isnan().all() and not both[0].isnan().any() and not both[2].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(2, 9000), (1100, 4096), (1100, 4103)])
@pytest.mark.parametrize("top", [32, 33, 64])
def test_rows_of_one_value_with_many_alternatives(dtype, rows, vocab, top):
    """All of a row equal, masked or NaN: as many equal logits as the search for
    the likeliest may meet, the first token among them."""
    logits = torch.randn(rows, vocab, device="cuda").to(dtype)
    logits[0] = float("nan")
    logits[1] = 0.0
    if rows > 2:
        logits[2, 1:] = -1.0
        logits[2, 0] = float("nan")
        logits[3] = float("-inf")
        logits[4, 40:] = float("-inf")
        logits[5] = torch.finfo(dtype).min
        logits[6, ::2] = float("nan")
        logits[7, :] = float("inf")
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    got = cf.token_logprobs(logits, tokens, 1.5, True, top)
    ref = reference(logits[:8], tokens[:8, None], 1.5, top)
    assert torch.equal(got.top_tokens[:8].cpu(), ref[3])
    close(got.top_logprobs[:8], ref[2], logprob_tolerance(ref[2], vocab))


@pytest.mark.parametrize("shape", [(), (3,), (1, 2), (2, 1, 1), (2, 0)])
def test_tokens_that_do_not_fit_are_refused_alike_on_the_gpu(shape):
    tokens = torch.zeros(shape, dtype=torch.int64, device="cuda")
    for logits in (torch.zeros(2, 100, device="cuda"), torch.zeros(2, 100, device="cuda", requires_grad=True)):
        with pytest.raises(ValueError):
            cf.token_logprobs(logits, tokens)


@pytest.mark.parametrize("top", [0, 64])
def test_the_longest_row_there_is(top):
    """2^27 floats: as many chunks as the join takes."""
    vocab = 2**27
    logits = torch.randn(1, vocab, device="cuda")
    peaks = torch.randperm(vocab, device="cuda")[:64]
    logits[0, peaks] = 40.0 - 0.25 * torch.arange(64, device="cuda")
    got = cf.token_logprobs(logits, peaks[None, :3].contiguous(), 1.0, True, top)
    if top:
        assert torch.equal(got.top_tokens[0], peaks)
    x = logits[0].double()
    logp = x - x.logsumexp(0)
    ref = logp[peaks[:3]][None].cpu()
    close(got.logprobs, ref, logprob_tolerance(ref, vocab // 1024))
    entropy = -(logp.exp() * logp).sum()[None].cpu()
    close(got.entropy, entropy, entropy_tolerance(entropy, vocab // 1024))


@pytest.mark.parametrize("rows", [255, 256, 257, 511, 512, 513, 1023, 1025])
@pytest.mark.parametrize("vocab,top", [(4103, 3), (66000, 9), (66000, 8)])
def test_rows_on_both_sides_of_where_they_are_cut(rows, vocab, top):
    logits = torch.randn(rows, vocab, device="cuda").bfloat16().requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device="cuda")
    got = cf.token_logprobs(logits, tokens, 0.9, True, top)
    g, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    grad, = torch.autograd.grad([got.logprobs, got.entropy], [logits], [g, h])
    at = torch.tensor([0, 1, rows // 2, rows - 1])
    ref = reference(logits[at], tokens[at, None], 0.9, top)
    close(got.logprobs[at, None], ref[0], logprob_tolerance(ref[0], vocab))
    close(got.entropy[at], ref[1], entropy_tolerance(ref[1], vocab))
    assert torch.equal(got.top_tokens[at].cpu(), ref[3])
    want, size = gradient(logits[at], tokens[at, None], 0.9, g[at, None], h[at])
    close(grad[at], want, 2.0**-8 * want.abs() + (2.0**-18 + 8 * 2.0**-24 * vocab / 256) * size + 2.0**-130)
