"""Decay attention against the float64 recurrence.

Tolerances, elementwise, from the arithmetic alone: a result r is a nested sum
of products; A is the same sum over absolute values. float32 sums of n terms
err by at most n 2^-24 A (n: the dot products' lengths, a chunk, and one
rounding per chunk for the carried state). bfloat16 operands are exact in
float32; the products a chunk forms before its second product carry two
bfloat16 terms (relative 2^-17 each, two of them in series), the products
added to the state three terms (2^-24); a bfloat16 result is rounded once
(2^-8 of a unit in the last place's binade: 2^-8 |r| covers half an ulp).
"""

import pytest
import torch

from oracle.decay import attention

pytestmark = pytest.mark.gpu


def _inputs(batch, time, heads, kv, dk, dv, dtype, seed=0, fused=False):
    g = torch.Generator().manual_seed(seed)
    shapes = ((heads, dk), (kv, dk), (kv, dv))
    if fused:
        proj = torch.randn(batch, time, sum(n * d for n, d in shapes), generator=g).to(dtype).cuda()
        parts = proj.split([n * d for n, d in shapes], dim=-1)
        qkv = [p.view(batch, time, n, d) for p, (n, d) in zip(parts, shapes)]
    else:
        qkv = [torch.randn(batch, time, n, d, generator=g).to(dtype).cuda() for n, d in shapes]
    decay = -torch.exp(torch.empty(heads).uniform_(-6.0, -0.5, generator=g)).cuda()
    initial = torch.randn(batch, heads, dk, dv, generator=g).cuda()
    return (*qkv, decay, initial)


def _tolerance(result, absolute, time, dk, dv, dtype, state):
    n = 2 * max(dk, dv) + 2 * 64 + 2 * (time // 64 + 1) + 16
    tol = n * 2.0 ** -24 * absolute
    if dtype == torch.bfloat16:
        tol = tol + (2.0 ** -22 if state else 2.0 ** -16) * absolute
        if not state:
            tol = tol + 2.0 ** -8 * result.abs()
    return tol + 1e-30


def _close(name, got, want, absolute, time, dk, dv, dtype, state=False):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    err = (got - want).abs()
    tol = _tolerance(want, absolute, time, dk, dv, dtype, state)
    assert bool((err <= tol).all()), (name, float((err / tol).max()))


def _compare(batch, time, heads, kv, dk, dv, dtype, lengths=None, with_initial=True, fused=False, seed=0):
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(batch, time, heads, kv, dk, dv, dtype, seed, fused)
    scale = dk ** -0.5
    init = initial if with_initial else None
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(seed + 1)
    d_out = torch.randn(batch, time, heads, dv, generator=g).to(dtype).cuda()
    d_fin = torch.randn(batch, heads, dk, dv, generator=g).cuda()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)] + ([init.requires_grad_(True)] if with_initial else [])
    res = decay_attention(leaves[0], leaves[1], leaves[2], decay, initial=leaves[3] if with_initial else None, lengths=lens)
    assert res.output.dtype == dtype and res.state.dtype == torch.float32
    grads = torch.autograd.grad((res.output, res.state), leaves, (d_out, d_fin))
    want = attention(q, k, v, decay, scale, init, lens, d_out, d_fin)
    a = lambda t: None if t is None else t.detach().abs()  # noqa: E731
    absolute = attention(a(q), a(k), a(v), decay, scale, a(init), lens, a(d_out), a(d_fin))
    args = (time, dk, dv, dtype)
    _close("output", res.output, want["output"], absolute["output"], *args)
    _close("state", res.state, want["state"], absolute["state"], *args, state=True)
    for name, got in zip(("dq", "dk", "dv"), grads):
        _close(name, got, want[name], absolute[name], *args)
    if with_initial:
        _close("d_initial", grads[3], want["d_initial"], absolute["d_initial"], *args, state=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("time", [1, 2, 63, 64, 65, 127, 200])
def test_lengths_around_a_chunk(dtype, time):
    _compare(2, time, 2, 2, 64, 64, dtype, seed=time)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(64, 128), (128, 64), (128, 128), (8, 8), (40, 72), (80, 96), (20, 7), (1, 1), (127, 121)])
def test_key_and_value_dims(dtype, dk, dv):
    _compare(2, 150, 3, 3, dk, dv, dtype, seed=dk + dv)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv", [(4, 1), (6, 2), (3, 3)])
def test_shared_heads_and_slices_of_one_projection(dtype, heads, kv):
    _compare(2, 100, heads, kv, 64, 128, dtype, fused=True, seed=heads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ragged_lengths(dtype):
    _compare(6, 130, 2, 1, 64, 64, dtype, lengths=[0, 1, 64, 65, 130, 500], seed=3)


def test_no_initial_state_and_a_longer_sequence():
    _compare(1, 1500, 2, 2, 64, 64, torch.bfloat16, with_initial=False, seed=4)


def test_one_row_over_many_chunks_equals_two_calls_with_a_carried_state():
    """A long sequence with few heads (the case a kernel may split over time)
    and the same sequence in two calls, the second from the first's state."""
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(1, 6000, 1, 1, 128, 128, torch.bfloat16, seed=5)
    decay = torch.full_like(decay, -0.002)
    whole = decay_attention(q, k, v, decay, initial=initial)
    first = decay_attention(q[:, :2500], k[:, :2500], v[:, :2500], decay, initial=initial)
    second = decay_attention(q[:, 2500:], k[:, 2500:], v[:, 2500:], decay, initial=first.state)
    a = [t.abs() for t in (q, k, v)]
    absolute = attention(*a, decay, 128 ** -0.5, initial.abs())
    joined = torch.cat((first.output, second.output), 1).double().cpu()
    _close("output", whole.output, joined, absolute["output"] * 2, 6000, 128, 128, torch.bfloat16)
    _close("state", whole.state, second.state.double().cpu(), absolute["state"] * 2, 6000, 128, 128, torch.bfloat16, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_places_past_a_length_are_never_read(dtype):
    """NaN and inf past the lengths: same results, finite gradients, zeros there."""
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(3, 100, 2, 2, 64, 128, dtype, seed=6)
    lens = torch.tensor([0, 37, 64], dtype=torch.int32, device="cuda")
    inside = (torch.arange(100, device="cuda") < lens[:, None])[:, :, None, None]
    clean = [torch.where(inside, t, 0.0) for t in (q, k, v)]
    dirty = [torch.where(inside, t, float("nan") if i % 2 else float("inf")) for i, t in enumerate((q, k, v))]
    d_out = torch.randn(3, 100, 2, 128, device="cuda").to(dtype)
    d_dirty = torch.where(inside, d_out, float("nan"))
    got = []
    for operands, d in ((clean, d_out), (dirty, d_dirty)):
        leaves = [t.detach().clone().requires_grad_(True) for t in operands]
        res = decay_attention(*leaves, decay, initial=initial, lengths=lens)
        got.append((res.output, res.state, *torch.autograd.grad(res.output, leaves, d)))
    for x, y in zip(*got):
        assert bool(torch.isfinite(y).all()) and torch.equal(x, y)
    assert not bool(got[1][0][~inside[..., 0, 0]].any())


def test_decay_extremes():
    """No decay (0), a decay that leaves only the own token (-inf), and one that underflows within a chunk."""
    from mamba4_b200 import decay_attention

    q, k, v, _, initial = _inputs(1, 200, 3, 3, 64, 64, torch.bfloat16, seed=7)
    decay = torch.tensor([0.0, float("-inf"), -3.0], device="cuda")
    res = decay_attention(q, k, v, decay, initial=initial)
    want = attention(q, k, v, decay, 0.125, initial)
    absolute = attention(q.abs(), k.abs(), v.abs(), decay, 0.125, initial.abs())
    _close("output", res.output, want["output"], absolute["output"], 200, 64, 64, torch.bfloat16)
    _close("state", res.state, want["state"], absolute["state"], 200, 64, 64, torch.bfloat16, True)


@pytest.mark.parametrize("operand", [0, 1, 2, 3])
def test_gradients_against_differences(operand):
    """The output is linear in each operand, so the difference of the loss at
    x + d and x - d is twice the gradient's product with d, for any d; float32,
    both sides sums with the bounds above (4 of them)."""
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(2, 90, 2, 2, 24, 40, torch.float32, seed=8)
    d_out, d_fin = torch.randn(2, 90, 2, 40, device="cuda"), torch.randn(2, 2, 24, 40, device="cuda")
    operands = [q, k, v, initial]

    def loss(x, sign):
        args = list(operands)
        args[operand] = x
        res = decay_attention(*args[:3], decay, initial=args[3])
        return float((res.output.double() * d_out).sum() + (res.state.double() * d_fin).sum()) * sign

    x = operands[operand]
    d = torch.randn_like(x)
    leaf = x.clone().requires_grad_(True)
    args = list(operands)
    args[operand] = leaf
    res = decay_attention(*args[:3], decay, initial=args[3])
    grad, = torch.autograd.grad((res.output, res.state), leaf, (d_out, d_fin))
    difference = (loss(x + d, 1) + loss(x - d, -1)) / 2
    a = attention(q.abs(), k.abs(), v.abs(), decay, 24 ** -0.5, initial.abs(), None, d_out.abs(), d_fin.abs())
    name = ("dq", "dk", "dv", "d_initial")[operand]
    size = float((a[name] * (x.abs() + d.abs()).double().cpu()).sum())
    assert abs(float((grad.double() * d).sum()) - difference) <= 4 * (2 * 40 + 128 + 20) * 2.0 ** -24 * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,heads,kv,dk,dv", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 128), (2, 3, 3, 20, 7), (5, 2, 1, 128, 100)])
def test_step_against_one_token_of_the_recurrence(dtype, batch, heads, kv, dk, dv):
    from mamba4_b200 import decay_attention_step

    q, k, v, decay, state = _inputs(batch, 1, heads, kv, dk, dv, dtype, seed=9)
    args = (state, q[:, 0], k[:, 0], v[:, 0], decay)
    res = decay_attention_step(*args)
    want = attention(q, k, v, decay, dk ** -0.5, state)
    absolute = attention(q.abs(), k.abs(), v.abs(), decay, dk ** -0.5, state.abs())
    _close("output", res.output[:, None], want["output"], absolute["output"], 1, dk, dv, dtype)
    _close("state", res.state, want["state"], absolute["state"], 1, dk, dv, torch.float32)
    held = state.clone()
    inplace = decay_attention_step(held, *args[1:], inplace=True)
    assert inplace.state.data_ptr() == held.data_ptr()
    assert torch.equal(held, res.state) and torch.equal(inplace.output, res.output)


def test_steps_continue_a_prompt():
    """A prompt through the chunked form, then tokens one by one, equal the whole through the chunked form."""
    from mamba4_b200 import decay_attention, decay_attention_step

    q, k, v, decay, _ = _inputs(2, 80, 2, 2, 64, 128, torch.float32, seed=10)
    whole = decay_attention(q, k, v, decay)
    res = decay_attention(q[:, :70], k[:, :70], v[:, :70], decay)
    state, outs = res.state, []
    for t in range(70, 80):
        step = decay_attention_step(state, q[:, t], k[:, t], v[:, t], decay)
        state = step.state
        outs.append(step.output)
    absolute = attention(q.abs(), k.abs(), v.abs(), decay, 0.125)
    _close("output", torch.stack(outs, 1), whole.output[:, 70:].double().cpu(), 2 * absolute["output"][:, 70:], 80, 64,
           128, torch.float32)
    _close("state", state, whole.state.double().cpu(), 2 * absolute["state"], 80, 64, 128, torch.float32)


def test_empty_batches_and_times():
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(2, 5, 2, 2, 16, 24, torch.bfloat16)
    res = decay_attention(q[:, :0], k[:, :0], v[:, :0], decay, initial=initial)
    assert res.output.shape == (2, 0, 2, 24) and torch.equal(res.state, initial)
    res = decay_attention(q[:0], k[:0], v[:0], decay)
    assert res.output.shape == (0, 5, 2, 24) and res.state.shape == (0, 2, 16, 24)


def test_another_stream():
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(2, 300, 2, 2, 64, 64, torch.bfloat16, seed=11)
    want = decay_attention(q, k, v, decay, initial=initial)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = decay_attention(q, k, v, decay, initial=initial)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)


def test_refusals():
    from mamba4_b200 import decay_attention, decay_attention_step

    q, k, v, decay, initial = _inputs(2, 5, 4, 2, 16, 24, torch.bfloat16)
    with pytest.raises(ValueError, match="dtype"):
        decay_attention(q.half(), k.half(), v.half(), decay)
    with pytest.raises(ValueError, match="dtype"):
        decay_attention(q, k.float(), v, decay)
    with pytest.raises(ValueError, match="multiple"):
        decay_attention(q[:, :, :3], k, v, decay[:3])
    with pytest.raises(ValueError, match="agree"):
        decay_attention(q, k[:, :4], v, decay)
    with pytest.raises(ValueError, match="1..128"):
        big = torch.zeros(1, 2, 1, 136, device="cuda")
        decay_attention(big, big, big, decay[:1])
    with pytest.raises(ValueError, match="log_decay"):
        decay_attention(q, k, v, decay[:3])
    with pytest.raises(ValueError, match="no gradient"):
        decay_attention(q, k, v, decay.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="initial"):
        decay_attention(q, k, v, decay, initial=initial[:1])
    with pytest.raises(ValueError, match="lengths"):
        decay_attention(q, k, v, decay, lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="state"):
        decay_attention_step(initial.double(), q[:, 0], k[:, 0], v[:, 0], decay)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dk,dv,kv", [(64, 64, 2), (64, 128, 1), (128, 64, 2), (128, 128, 1), (40, 72, 2), (80, 96, 1)])
def test_not_a_number_reaches_later_tokens_only(dtype, dk, dv, kv):
    """A NaN or an infinity at one place of an operand: what does not depend on
    it in the recurrence is as without it, the rest is not finite."""
    from mamba4_b200 import decay_attention

    nan, inf = float("nan"), float("inf")
    places = [("v", 37, nan), ("v", 63, inf), ("v", 64, -inf), ("k", 70, inf), ("k", 1, nan), ("q", 100, nan),
              ("d", 37, nan), ("d", 64, inf), ("v", 149, nan), ("k", 127, -inf), ("d", 149, nan), ("q", 0, inf)]
    batch, time, heads = len(places), 150, 2
    q, k, v, decay, initial = _inputs(batch, time, heads, kv, dk, dv, dtype, seed=dk + dv)
    d_out = torch.randn(batch, time, heads, dv, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    clean = dict(q=q, k=k, v=v, d=d_out)
    bad = {n: x.clone() for n, x in clean.items()}
    for row, (name, t, value) in enumerate(places):
        x = bad[name]
        x[row, t, -1, 5 * row % x.shape[-1]] = value
        clean[name][row, t, -1, 5 * row % x.shape[-1]] = 0.0
    leaves = [bad[n].requires_grad_(True) for n in "qkv"] + [initial.requires_grad_(True)]
    res = decay_attention(*leaves[:3], decay, initial=leaves[3])
    got = dict(output=res.output, state=res.state)
    got.update(zip(("dq", "dk", "dv", "d_initial"), torch.autograd.grad(res.output, leaves, bad["d"])))
    scale = dk ** -0.5
    want = attention(*(bad[n] for n in "qkv"), decay, scale, initial, None, bad["d"])
    absolute = attention(*(clean[n].abs() for n in "qkv"), decay, scale, initial.abs(), None, clean["d"].abs())
    for name, w in want.items():
        x, state = got[name].detach().double().cpu(), name in ("state", "d_initial")
        finite = torch.isfinite(w)
        assert torch.equal(torch.isfinite(x), finite), (name, torch.nonzero(torch.isfinite(x) != finite)[:3].tolist())
        tol = _tolerance(w, absolute[name], time, dk, dv, dtype, state)
        assert bool(((x - w).abs() <= tol)[finite].all()), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dk,dv,kv,time", [(64, 64, 1, 100), (64, 128, 2, 100), (128, 64, 1, 100), (128, 128, 2, 100), (40, 72, 1, 1100)])
def test_zeros_past_a_length_whatever_the_state_holds(dtype, dk, dv, kv, time):
    """States that are not finite: outputs and gradients past a length are zero all the same."""
    from mamba4_b200 import decay_attention

    lens = torch.tensor([0, 37, 64, 90], dtype=torch.int32, device="cuda")
    q, k, v, decay, initial = _inputs(4, time, 2, kv, dk, dv, dtype, seed=dk + dv)
    outside = torch.arange(time, device="cuda") >= lens[:, None]
    for bad in (float("nan"), float("inf"), float("-inf")):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        initial[:, :, ::3, ::2] = bad
        res = decay_attention(*leaves, decay, initial=initial, lengths=lens)
        grads = torch.autograd.grad((res.output, res.state), leaves, (torch.randn_like(res.output), initial))
        for x in (res.output, *grads):
            assert not bool(x.detach()[outside].any())
            assert not bool(torch.isfinite(x.detach()[~outside]).all())


@pytest.mark.parametrize("operand", [0, 1, 2, 3])
def test_forward_mode_is_refused(operand):
    from torch.autograd import forward_ad
    from mamba4_b200 import decay_attention

    args = list(_inputs(1, 5, 1, 1, 8, 8, torch.float32))
    args[3], decay = args[4], args[3]
    with forward_ad.dual_level():
        args[operand] = forward_ad.make_dual(args[operand], torch.ones_like(args[operand]))
        with pytest.raises(NotImplementedError):
            decay_attention(*args[:3], decay, initial=args[3])


def test_second_derivatives_are_refused():
    from mamba4_b200 import decay_attention

    q, k, v, decay, _ = _inputs(1, 5, 1, 1, 8, 8, torch.float32)
    q.requires_grad_(True)
    grad, = torch.autograd.grad(decay_attention(q, k, v, decay).output.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(20, 7), (3, 16), (64, 65)])
def test_a_state_of_odd_dims_goes_on_in_place(dtype, dk, dv):
    from mamba4_b200 import decay_attention, decay_attention_step

    q, k, v, decay, initial = _inputs(2, 30, 2, 1, dk, dv, dtype, seed=22)
    state = decay_attention(q[:, :29], k[:, :29], v[:, :29], decay, initial=initial).state
    assert state.is_contiguous()
    step = decay_attention_step(state, q[:, 29], k[:, 29], v[:, 29], decay, inplace=True)
    whole = decay_attention(q, k, v, decay, initial=initial)
    absolute = attention(q.abs(), k.abs(), v.abs(), decay, dk ** -0.5, initial.abs())
    _close("state", step.state, whole.state.double().cpu(), 2 * absolute["state"], 30, dk, dv, dtype, True)
    across = initial.transpose(2, 3).contiguous().transpose(2, 3)
    assert decay_attention(q[:, :0], k[:, :0], v[:, :0], decay, initial=across).state.is_contiguous()


def test_a_state_updated_in_place_is_noticed():
    """A backward pass that needs the state as it was before the update fails."""
    from mamba4_b200 import decay_attention, decay_attention_step

    q, k, v, decay, state = _inputs(1, 6, 1, 1, 8, 8, torch.float32, seed=23)
    q.requires_grad_(True)
    out = decay_attention(q, k, v, decay, initial=state).output
    with torch.no_grad():
        decay_attention_step(state, q[:, 0], k[:, 0], v[:, 0], decay, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():
        held = state.clone()
        decay_attention_step(held, q[:, 0], k[:, 0], v[:, 0], decay, inplace=True)
    with torch.no_grad():
        decay_attention_step(held, q[:, 0], k[:, 0], v[:, 0], decay, inplace=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lengths_of_64_bits(dtype):
    """Values past T count as T before they are narrowed to 32 bits."""
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(4, 70, 2, 2, 16, 24, dtype, seed=21)
    got = decay_attention(q, k, v, decay, initial=initial,
                          lengths=torch.tensor([2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 40], device="cuda"))
    want = decay_attention(q, k, v, decay, initial=initial,
                           lengths=torch.tensor([70, 70, 70, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
    for narrow in (torch.uint8, torch.int16, torch.bool):
        some = torch.tensor([1, 0, 1, 1], device="cuda")
        x, y = (decay_attention(q, k, v, decay, lengths=n).output for n in (some.to(narrow), some.int()))
        assert torch.equal(x, y)


def test_empty_axes_have_gradients():
    from mamba4_b200 import decay_attention

    q, k, v, decay, initial = _inputs(2, 5, 2, 2, 16, 24, torch.bfloat16)
    for cut in (lambda t: t[:, :0], lambda t: t[:0]):
        leaves = [cut(t).detach().requires_grad_(True) for t in (q, k, v)]
        out = decay_attention(*leaves, decay).output
        for leaf, grad in zip(leaves, torch.autograd.grad(out, leaves, torch.zeros_like(out))):
            assert grad.shape == leaf.shape
        leaves.append(initial[:leaves[0].shape[0]].detach().requires_grad_(True))
        res = decay_attention(*leaves[:3], decay, initial=leaves[3])
        grads = torch.autograd.grad((res.output, res.state), leaves, (torch.zeros_like(res.output), leaves[3].detach()))
        assert torch.equal(grads[3], leaves[3]) and grads[2].shape == leaves[2].shape
        assert torch.autograd.grad(decay_attention(*leaves[:3], decay, initial=leaves[3]).output.sum(), leaves)[3].abs().sum() == 0


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (80, 96)])
@pytest.mark.parametrize("lengths", [None, [1100, 300], [0, 777]])
def test_segments_of_the_time_axis(dk, dv, lengths):
    """Few heads over many chunks are walked in segments, in both directions;
    slow decays carry over several of them."""
    from mamba4_b200 import decay_attention

    dtype, time = torch.bfloat16, 1100
    q, k, v, decay, initial = _inputs(2, time, 2, 1, dk, dv, dtype, seed=dk + 2 * dv)
    decay = torch.tensor([-0.002, -0.0005], device="cuda")
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(2)
    d_out = torch.randn(2, time, 2, dv, generator=g).to(dtype).cuda()
    d_fin = torch.randn(2, 2, dk, dv, generator=g).cuda()
    leaves = [t.requires_grad_(True) for t in (q, k, v, initial)]
    res = decay_attention(*leaves[:3], decay, initial=initial, lengths=lens)
    got = dict(output=res.output, state=res.state)
    got.update(zip(("dq", "dk", "dv", "d_initial"), torch.autograd.grad((res.output, res.state), leaves, (d_out, d_fin))))
    scale = dk ** -0.5
    want = attention(q, k, v, decay, scale, initial, lens, d_out, d_fin)
    a = [t.detach().abs() for t in (q, k, v, initial, d_out, d_fin)]
    absolute = attention(*a[:3], decay, scale, a[3], lens, *a[4:])
    for name, x in got.items():
        _close(name, x, want[name], absolute[name], time, dk, dv, dtype, state=name in ("state", "d_initial"))


@pytest.mark.parametrize("batch,heads", [(4, 12), (40, 8)])
def test_float32_walks_of_more_columns_a_block(batch, heads):
    _compare(batch, 70, heads, heads, 24, 72, torch.float32, lengths=[70 - i for i in range(batch)], seed=24)


@pytest.mark.parametrize("dk,dv,kv", [(64, 64, 1), (64, 128, 2), (128, 128, 1)])
def test_not_a_number_in_a_segment(dk, dv, kv):
    """Walks in segments, with lengths and final-state gradients: as in one."""
    from mamba4_b200 import decay_attention

    dtype, time, nan = torch.bfloat16, 1100, float("nan")
    q, k, v, decay, initial = _inputs(2, time, 2, kv, dk, dv, dtype, seed=dk)
    decay = torch.tensor([-0.002, -0.01], device="cuda")
    lens = torch.tensor([1000, 777], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(3)
    d_out = torch.randn(2, time, 2, dv, generator=g).to(dtype).cuda()
    d_fin = torch.randn(2, 2, dk, dv, generator=g).cuda()
    k[0, 300, -1, 3] = v[1, 520, -1, 2] = d_out[0, 700, -1, 5] = nan
    leaves = [t.requires_grad_(True) for t in (q, k, v, initial)]
    res = decay_attention(*leaves[:3], decay, initial=initial, lengths=lens)
    got = dict(output=res.output, state=res.state)
    got.update(zip(("dq", "dk", "dv", "d_initial"), torch.autograd.grad((res.output, res.state), leaves, (d_out, d_fin))))
    want = attention(q, k, v, decay, dk ** -0.5, initial, lens, d_out, d_fin)
    a = [torch.nan_to_num(t.detach()).abs() for t in (q, k, v, initial, d_out, d_fin)]
    absolute = attention(*a[:3], decay, dk ** -0.5, a[3], lens, *a[4:])
    for name, w in want.items():
        x, finite = got[name].detach().double().cpu(), torch.isfinite(w)
        assert torch.equal(torch.isfinite(x), finite), name
        tol = _tolerance(w, absolute[name], time, dk, dv, dtype, name in ("state", "d_initial"))
        assert bool(((x - w).abs() <= tol)[finite].all()), name


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (80, 96)])
def test_carried_states_hold_32_bits(dk, dv):
    """Two tokens whose contributions to a carried state cancel but for the decay
    of one token, e^g = 1 - 2^-12: what is left is 2^-12 of each, so that the
    result has 12 bits less than the contributions had. Each of those is a product
    of the scale, an exponential (2 ulp), a power of the decay and two operands,
    rounded at most 8 times to 24 bits (2^-21 of the absolute sum); the bfloat16
    result is rounded once."""
    from mamba4_b200 import decay_attention

    time, dtype = 192, torch.bfloat16
    q, k, v, _, _ = _inputs(2, time, 2, 2, dk, dv, dtype, seed=dk + dv)
    d_out = torch.randn(2, time, 2, dv, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    decay = torch.full((2,), -2.0 ** -12, device="cuda")

    def pair(x, y, at):
        x, y = (torch.zeros_like(t).index_copy_(1, torch.tensor([at, at + 1], device="cuda"), t[:, [at, at]]) for t in (x, y))
        y[:, at + 1] *= -1
        return x, y

    for name, args in (("dk", (*pair(q, d_out, 130), k, v)), ("dq", (q, d_out, *pair(k, v, 10)))):
        q1, d1, k1, v1 = args
        leaves = [t.detach().requires_grad_(True) for t in (q1, k1, v1)]
        grads = torch.autograd.grad(decay_attention(*leaves, decay).output, leaves, d1)
        want = attention(q1, k1, v1, decay, dk ** -0.5, None, None, d1)[name]
        absolute = attention(q1.abs(), k1.abs(), v1.abs(), decay, dk ** -0.5, None, None, d1.abs())[name]
        part = slice(0, 128) if name == "dk" else slice(64, None)
        err = (grads[name == "dk"].double().cpu() - want)[:, part].abs()
        tol = (2.0 ** -8 * want.abs() + 2.0 ** -21 * absolute)[:, part] + 1e-30
        assert bool((err <= tol).all()), (name, float((err / tol).max()))
