"""Embedding lookup and its gradient against float64.

Tolerances: the lookup rounds scale * w once in float32 and once to the output
type (2^-24 and, for bfloat16, 2^-9 relative, doubled for the double rounding).
The gradient is a float32 sum of n rows, at most n 2^-24 of the sum of absolute
values, times a scale (2^-24), rounded to the weight's type."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23


def _check(tokens, vocab, dim, weight_dtype, out_dtype, scale=3.7, seed=0):
    from mamba4_b200 import embedding_lookup

    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(vocab, dim, generator=g).to(weight_dtype).cuda().requires_grad_(True)
    grad = torch.randn(*tokens.shape, dim, generator=g).to(out_dtype).cuda()
    out = embedding_lookup(tokens.cuda(), weight, scale=scale, dtype=out_dtype)
    d_weight, = torch.autograd.grad(out, weight, grad)
    assert out.dtype == out_dtype and out.shape == (*tokens.shape, dim) and d_weight.dtype == weight_dtype
    flat = tokens.reshape(-1).long()
    inside = (flat >= 0) & (flat < vocab)
    w64, g64 = weight.detach().double().cpu(), grad.double().cpu().reshape(-1, dim)
    want = torch.zeros(flat.numel(), dim, dtype=torch.float64)
    want[inside] = scale * w64[flat[inside]]
    err = (out.detach().double().cpu().reshape(-1, dim) - want).abs()
    assert bool((err <= _unit(out_dtype) * want.abs() + 2.0 ** -23 * want.abs()).all())
    sums, sizes = torch.zeros(vocab, dim, dtype=torch.float64), torch.zeros(vocab, dim, dtype=torch.float64)
    sums.index_add_(0, flat[inside], g64[inside])
    sizes.index_add_(0, flat[inside], g64[inside].abs())
    counts = torch.bincount(flat[inside], minlength=vocab).double()[:, None]
    err = (d_weight.double().cpu() - scale * sums).abs()
    tol = scale * (counts + 2) * 2.0 ** -24 * sizes + _unit(weight_dtype) * scale * sums.abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    assert not bool(d_weight.cpu()[counts[:, 0] == 0].any())
    again, = torch.autograd.grad(embedding_lookup(tokens.cuda(), weight, scale=scale, dtype=out_dtype), weight, grad)
    assert torch.equal(again, d_weight)


@pytest.mark.parametrize("weight_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,dim", [(1, 1, 1), (5, 97, 64), (1024, 50, 24), (1025, 3000, 264), (3000, 40000, 20)])
def test_types_and_sizes(weight_dtype, out_dtype, rows, vocab, dim):
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(rows))
    _check(tokens, vocab, dim, weight_dtype, out_dtype, seed=rows + dim)


@pytest.mark.parametrize("count", [1, 63, 64, 65, 128, 129, 2048, 2049, 5000])
def test_one_id_many_times(count):
    """Runs around the piece size and past what one block holds in shared memory."""
    tokens = torch.full((count + 40,), 700)
    tokens[::7] = torch.randint(0, 1000, (tokens[::7].numel(),), generator=torch.Generator().manual_seed(count))
    _check(tokens, 1000, 72, torch.float32, torch.bfloat16, seed=count)


def test_skewed_ids_in_two_axes():
    g = torch.Generator().manual_seed(1)
    rank = torch.exp(torch.rand(8, 900, generator=g) * 9.0).long().clamp(max=8099)
    _check(rank, 8100, 96, torch.float32, torch.bfloat16)


def test_ids_outside_the_table():
    """Padding ids give zero rows and no gradient, in every combination with real ones."""
    tokens = torch.tensor([-1, 0, 11, 12, -100, 5, 5, 2 ** 40, -(2 ** 40)])
    _check(tokens, 12, 16, torch.float32, torch.float32)
    _check(torch.full((70,), -1), 12, 16, torch.float32, torch.bfloat16)


def test_int32_ids_and_rows_that_are_not_aligned():
    from mamba4_b200 import embedding_lookup

    weight = torch.randn(33 * 8 + 1, device="cuda")[1:].view(33, 8).requires_grad_(True)
    tokens = torch.randint(0, 33, (50,), device="cuda", dtype=torch.int32)
    out = embedding_lookup(tokens, weight)
    assert torch.equal(out.detach(), weight.detach()[tokens.long()])
    d, = torch.autograd.grad(out, weight, torch.ones_like(out))
    assert torch.equal(d[:, 0], torch.bincount(tokens.long(), minlength=33).float())


def test_a_gradient_against_differences():
    """The lookup is linear in the table: a difference along d equals the gradient's product with d."""
    from mamba4_b200 import embedding_lookup

    weight, d = torch.randn(40, 24, device="cuda"), torch.randn(40, 24, device="cuda")
    tokens, grad = torch.randint(0, 40, (300,), device="cuda"), torch.randn(300, 24, device="cuda")
    leaf = weight.clone().requires_grad_(True)
    got, = torch.autograd.grad(embedding_lookup(tokens, leaf, scale=2.0), leaf, grad)
    rows = lambda w: (embedding_lookup(tokens, w, scale=2.0).double() * grad).sum()  # noqa: E731
    difference = float(rows(weight + d) - rows(weight - d)) / 2
    size = float((2 * grad.abs().double() * (weight.abs() + d.abs())[tokens]).sum())
    assert abs(float((got.double() * d).sum()) - difference) <= 300 * 2.0 ** -24 * size


def test_empty_tokens():
    from mamba4_b200 import embedding_lookup

    weight = torch.randn(7, 16, device="cuda", requires_grad=True)
    out = embedding_lookup(torch.zeros(3, 0, dtype=torch.int64, device="cuda"), weight, dtype=torch.bfloat16)
    assert out.shape == (3, 0, 16) and out.dtype == torch.bfloat16
    d, = torch.autograd.grad(out, weight, torch.zeros_like(out))
    assert not bool(d.any())


def test_refusals():
    from mamba4_b200 import embedding_lookup

    weight, tokens = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="CUDA"):
        embedding_lookup(tokens.cpu(), weight)
    with pytest.raises(ValueError, match="tokens"):
        embedding_lookup(tokens.float(), weight)
    with pytest.raises(ValueError, match="weight"):
        embedding_lookup(tokens, weight.half())
    with pytest.raises(ValueError, match="weight"):
        embedding_lookup(tokens, weight[0])
    with pytest.raises(ValueError, match="output"):
        embedding_lookup(tokens, weight, dtype=torch.float16)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    from mamba4_b200 import embedding_lookup

    weight, tokens = torch.randn(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            embedding_lookup(tokens, forward_ad.make_dual(weight, torch.ones_like(weight)))


def test_second_derivatives_are_refused():
    from mamba4_b200 import embedding_lookup

    weight, tokens = torch.randn(5, 8, device="cuda", requires_grad=True), torch.zeros(3, dtype=torch.int64, device="cuda")
    grad, = torch.autograd.grad(embedding_lookup(tokens, weight).square().sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


def test_sizes_without_a_gradient_are_refused_at_the_call():
    """What the backward pass cannot take is said before the forward pass runs."""
    from mamba4_b200 import embedding_lookup

    weight = torch.zeros((1 << 21) + 1, 1, device="cuda")
    tokens = torch.tensor([1 << 21], device="cuda")
    assert embedding_lookup(tokens, weight).shape == (1, 1)
    with pytest.raises(ValueError, match="vocabular"):
        embedding_lookup(tokens, weight.requires_grad_(True))
    with pytest.raises(ValueError, match="tokens"):
        embedding_lookup(tokens.expand((1 << 28) + 1), torch.zeros(4, 1, device="cuda", requires_grad=True))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [260, 512, 520, 768, 776, 1024, 1030, 1600])
def test_wide_rows(out_dtype, dim):
    """Widths of one, two and three vectors a thread and of several sweeps; runs
    for one warp, for a block and in pieces."""
    g = torch.Generator().manual_seed(dim)
    tokens = torch.cat([torch.full((n,), 11 * n % 97) for n in (1, 3, 4, 5, 8, 40, 64, 65, 129, 400)])
    tokens = torch.cat((tokens, torch.randint(-1, 97, (300,), generator=g)))
    _check(tokens[torch.randperm(tokens.numel(), generator=g)], 97, dim, torch.float32, out_dtype, seed=dim)


def test_more_tiles_than_threads():
    """Over 262,144 tokens, the sort's block takes its tiles in several rounds."""
    tokens = torch.randint(-1, 700, (263000,), generator=torch.Generator().manual_seed(5))
    tokens[tokens > 600] = 5
    _check(tokens, 700, 8, torch.float32, torch.bfloat16)
