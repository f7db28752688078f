"""Token sampling against float64 and against exact integer arithmetic."""

import pytest
import torch

from oracle.sampling import row as exact_row

pytestmark = pytest.mark.gpu


def _plain(logits, uniform, temperature, top_k, top_p, min_p):
    """The definition in torch operations: float32 z, 64-bit integer masses, a full sort."""
    rows, vocab = logits.shape
    x = logits.float()
    x = torch.where(torch.isnan(x), -torch.inf, x)
    top = x.amax(-1, keepdim=True)
    greedy = ~(temperature > 0)[:, None]
    z = torch.where(x == top, 0.0, torch.where(x == -torch.inf, torch.inf,
                                               (top - x) * torch.where(greedy, 1.0, 1.0 / temperature[:, None])))
    e = torch.exp(-z)
    mass = (e * 2.0 ** 35).to(torch.int64)
    order = torch.sort(z, dim=-1, stable=True).indices
    s, es = mass.gather(-1, order), e.gather(-1, order)
    rank = torch.arange(vocab, device=x.device)
    k = torch.where(top_k > 0, top_k, vocab)[:, None]
    one = greedy | ~(top_p > 0)[:, None] | ~(min_p <= 1)[:, None]
    keep = rank < torch.where(one, 1, k)
    running = torch.cumsum(s * keep, -1)
    limit = torch.ceil(top_p.double().clamp(0, 1)[:, None] * running[:, -1:].double()).to(torch.int64)
    keep = keep & ((running - s < limit) | (top_p >= 1)[:, None] | (rank == 0)) & ((es >= min_p[:, None]) | (rank == 0))
    kept = torch.zeros_like(mass).scatter(-1, order, s * keep)
    running = torch.cumsum(kept, -1)
    total = running[:, -1:]
    target = torch.minimum((uniform[:, None].double() * total.double()).floor().to(torch.int64).clamp(min=0), total - 1)
    token = (running <= target).sum(-1)
    return torch.where(top[:, 0] == -torch.inf, -1, token), keep.sum(-1)


def _settings(rows, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)].cuda()  # noqa: E731
    return dict(temperature=pick([0.0, 0.5, 0.9, 1.0, 1.7]), top_k=pick([0, 1, 2, 40, 300, 10 ** 6]).to(torch.int32),
                top_p=pick([1.0, 0.99, 0.9, 0.5, 0.01]), min_p=pick([0.0, 0.0, 0.05, 0.5]))


def _exact_check(logits, uniform, settings, tokens, log_prob):
    """Float32 z carries 2 roundings of a value below 104 (beyond it e^-z
    underflows): relative 104 2^-22 < 3e-5 in a probability, and as much in the
    limits. The drawn token's interval of the running sum has to hold u within that."""
    slack = 3e-5
    for r in range(logits.shape[0]):
        args = [float(settings[n][r]) for n in ("temperature", "top_k", "top_p", "min_p")]
        low, high = exact_row(logits[r], float(uniform[r]), args[0], int(args[1]), args[2], args[3], slack)
        t, u = int(tokens[r]), float(uniform[r])
        assert high[t] > 0, (r, t)
        below, upto = float(high[:t].sum() / low.sum()), float(low[:t + 1].sum() / high.sum())
        least = float(low[:t].sum() / high.sum())
        most = float(high[:t + 1].sum() / low.sum())
        assert least * (1 - 2 * slack) - slack <= u <= most * (1 + 2 * slack) + slack, (r, t, below, upto, u)
        lp = float(log_prob[r])
        p = float(high[t])
        bounds = sorted((p / float(low.sum()), p / float(high.sum())))
        assert torch.log(torch.tensor(bounds[0])) - 1e-4 <= lp <= torch.log(torch.tensor(bounds[1])) + 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 33), (7, 1000), (4, 8192), (6, 8193), (5, 50304), (3, 70001), (2, 131072), (2, 200003), (1, 262144)])
def test_equal_to_the_definition(dtype, rows, vocab):
    from mamba4_b200 import sample_tokens

    g = torch.Generator().manual_seed(vocab)
    for repeat in range(4):
        logits = (3.0 * torch.randn(rows, vocab, generator=g)).to(dtype).cuda()
        if repeat == 3:
            logits[:, torch.rand(vocab, generator=g) < 0.7] = -torch.inf
            logits[:, vocab // 2] = 1.0
        uniform = torch.rand(rows, generator=g).cuda()
        settings = _settings(rows, vocab + repeat)
        got = sample_tokens(logits, uniform, **settings)
        want, _ = _plain(logits, uniform, **settings)
        assert torch.equal(got.tokens, want), (repeat, settings)
        _exact_check(logits, uniform, settings, got.tokens, got.log_prob)


def test_numbers_for_settings_equal_tensors():
    from mamba4_b200 import sample_tokens

    logits, uniform = 2 * torch.randn(9, 5000, device="cuda"), torch.rand(9, device="cuda")
    one = sample_tokens(logits, uniform, temperature=0.7, top_k=30, top_p=0.8, min_p=0.01)
    full = lambda v, d: torch.full((9,), v, device="cuda", dtype=d)  # noqa: E731
    per_row = sample_tokens(logits, uniform, temperature=full(0.7, torch.float32), top_k=full(30, torch.int64),
                            top_p=full(0.8, torch.float32), min_p=torch.tensor([0.01], device="cuda"))
    assert torch.equal(one.tokens, per_row.tokens) and torch.equal(one.log_prob, per_row.log_prob)


@pytest.mark.parametrize("vocab", [3000, 50304, 131072])
def test_equal_logits(vocab):
    """Every token ties: rank is by index; the boundary lies among more ties than any shared list holds."""
    from mamba4_b200 import sample_tokens

    logits = torch.full((8, vocab), -2.5, device="cuda")
    uniform = torch.tensor([0.0, 0.25, 0.5, 0.999999, 0.3, 0.7, 0.1, 0.9], device="cuda")
    settings = dict(temperature=torch.ones(8, device="cuda"),
                    top_k=torch.tensor([0, 0, 0, 0, 2000, 2000, 0, 2500], dtype=torch.int32, device="cuda"),
                    top_p=torch.tensor([1, 1, 1, 1, 1, 0.5, 0.7, 0.9], device="cuda"),
                    min_p=torch.zeros(8, device="cuda"))
    got = sample_tokens(logits, uniform, **settings)
    want, kept = _plain(logits, uniform, **settings)
    assert torch.equal(got.tokens, want)
    assert torch.allclose(got.log_prob, -torch.log(kept.float()), rtol=1e-6, atol=1e-6)


def test_crowded_values():
    """Tens of thousands of logits within a few float steps of each other: sub-histograms down to single values."""
    from mamba4_b200 import sample_tokens

    g = torch.Generator().manual_seed(3)
    steps = torch.randint(0, 40, (4, 60000), generator=g)
    logits = (10.0 - steps * 2.0 ** -20).cuda()
    logits[:, 17] = 11.0
    logits[2] = 0.125 * torch.randint(0, 3, (60000,), generator=g).cuda()
    logits[3] = logits[3] * 0 + 1e-30 * steps[3].cuda()
    uniform = torch.rand(4, generator=g).cuda()
    for k, p in ((0, 0.5), (30000, 1.0), (30000, 0.3), (45000, 0.9999), (7, 0.9)):
        settings = dict(temperature=torch.ones(4, device="cuda"), top_k=torch.full((4,), k, dtype=torch.int32, device="cuda"),
                        top_p=torch.full((4,), p, device="cuda"), min_p=torch.zeros(4, device="cuda"))
        got = sample_tokens(logits, uniform, **settings)
        want, _ = _plain(logits, uniform, **settings)
        assert torch.equal(got.tokens, want), (k, p)


def test_top_k_in_the_massless_tail():
    """top_k reaches tokens whose mass is zero, and more -inf logits than it keeps others."""
    from mamba4_b200 import sample_tokens

    logits = torch.linspace(0, -4000, 20000, device="cuda")[None].repeat(3, 1)
    logits[1, 100:] = -torch.inf
    logits[2] = -3.4e38
    logits[2, 5] = -3.3e38
    uniform = torch.tensor([0.5, 0.9, 0.999], device="cuda")
    settings = dict(temperature=torch.ones(3, device="cuda"), top_k=torch.full((3,), 15000, dtype=torch.int32, device="cuda"),
                    top_p=torch.tensor([0.9, 1.0, 0.95], device="cuda"), min_p=torch.zeros(3, device="cuda"))
    got = sample_tokens(logits, uniform, **settings)
    want, _ = _plain(logits, uniform, **settings)
    assert torch.equal(got.tokens, want)


def test_rows_a_mask_leaves_empty_and_special_values():
    from mamba4_b200 import sample_tokens

    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[-inf] * 4, [nan, -inf, nan, -inf], [nan, 1.0, 1.0, -inf], [inf, 0.0, inf, 1.0],
                           [low] * 4, [low, low, 0.0, low]], device="cuda")
    uniform = torch.tensor([0.5, 0.5, 0.6, 0.6, 0.6, 0.999], device="cuda")
    got = sample_tokens(logits, uniform, temperature=0.5)
    assert got.tokens.tolist() == [-1, -1, 2, 2, 2, 2]
    want = torch.log(torch.tensor([0.0, 0.0, 0.5, 0.5, 0.25, 1.0]))
    assert torch.allclose(got.log_prob.cpu(), want, rtol=1e-6, atol=1e-6)
    greedy = sample_tokens(logits, uniform, temperature=0.0)
    assert greedy.tokens.tolist() == [-1, -1, 1, 0, 0, 2] and greedy.log_prob.tolist()[2:] == [0.0] * 4


def test_settings_at_their_ends():
    """NaN and out-of-range settings leave the first-ranked token or switch a filter off; numbers outside [0, 1) clamp."""
    from mamba4_b200 import sample_tokens

    logits = torch.tensor([[0.0, 3.0, 1.0, 3.0]], device="cuda").repeat(8, 1)
    t = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    nan = float("nan")
    got = sample_tokens(logits, t(0.99, 0.99, 0.99, 0.99, 0.99, -1.0, 2.0, nan), temperature=t(nan, -1., 1., 1., 1., 1., 1., 1.),
                        top_k=t(0, 0, 0, 0, -5, 0, 0, 0).int(), top_p=t(1., 1., 0., nan, 1., 2., 2., 1.),
                        min_p=t(0., 0., 0., 0., 2., -1., 0., 0.))
    assert got.tokens.tolist() == [1, 1, 1, 1, 1, 0, 3, 0]


def test_strided_rows_and_leading_axes():
    from mamba4_b200 import sample_tokens

    wide = torch.randn(6, 1037, device="cuda")
    uniform = torch.rand(6, device="cuda")
    want = sample_tokens(wide[:, 3:1003].contiguous(), uniform, top_p=0.9)
    for logits in (wide[:, 3:1003], wide[:, 3:1003].t().contiguous().t()):
        got = sample_tokens(logits, uniform, top_p=0.9)
        assert torch.equal(got.tokens, want.tokens)
    got = sample_tokens(wide[:, 3:1003].reshape(2, 3, 1000), uniform.view(2, 3), top_p=0.9)
    assert torch.equal(got.tokens, want.tokens.view(2, 3)) and got.log_prob.shape == (2, 3)
    flat = sample_tokens(wide[0, 3:1003], uniform[0], top_p=0.9)
    assert flat.tokens.shape == () and int(flat.tokens) == int(want.tokens[0])
    empty = sample_tokens(wide[:0], uniform[:0])
    assert empty.tokens.shape == (0,)


def test_frequencies():
    """20000 draws from 6 tokens: each frequency within 5 standard deviations (2 in 10^6 by chance)."""
    from mamba4_b200 import sample_tokens

    n = 20000
    logits = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -3.0], device="cuda")
    g = torch.Generator().manual_seed(0)
    got = sample_tokens(logits.repeat(n, 1), torch.rand(n, generator=g).cuda(), temperature=1.5)
    p = torch.softmax(logits.double().cpu() / 1.5, 0)
    share = torch.bincount(got.tokens.cpu(), minlength=6).double() / n
    assert bool(((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all())


def test_refusals():
    from mamba4_b200 import sample_tokens

    logits, uniform = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(RuntimeError, match="CUDA"):
        sample_tokens(logits.cpu(), uniform)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        sample_tokens(logits.double(), uniform)
    with pytest.raises(ValueError, match="uniform"):
        sample_tokens(logits, uniform[:1])
    with pytest.raises(ValueError, match="vocabulary"):
        sample_tokens(torch.zeros(1, 262145, device="cuda"), uniform[:1])
    with pytest.raises(ValueError, match="top_p"):
        sample_tokens(logits, uniform, top_p=torch.ones(3, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [50304, 131072])
def test_places_unlike_each_other(dtype, vocab):
    """One place in four is 1 or 6 higher or lower than the others, for each of
    the places: what part of a row suggests about the boundary is wrong."""
    from mamba4_b200 import sample_tokens

    g = torch.Generator().manual_seed(vocab)
    logits, shifts = torch.randn(16, vocab, generator=g), [(p, d) for p in range(4) for d in (-6.0, -1.0, 1.0, 6.0)]
    for r, (place, shift) in enumerate(shifts):
        logits[r, place::4] += shift
    logits = logits.to(dtype).cuda()
    for repeat, (k, p) in enumerate([(0, 0.9), (0, 0.999), (1500, 0.8), (20000, 0.95), (vocab - 7, 1.0)]):
        uniform = torch.rand(16, generator=g).cuda()
        settings = dict(temperature=torch.ones(16, device="cuda"),
                        top_k=torch.full((16,), k, dtype=torch.int32, device="cuda"),
                        top_p=torch.full((16,), p, device="cuda"),
                        min_p=torch.full((16,), 1e-4 * (repeat % 2), device="cuda"))
        got = sample_tokens(logits, uniform, **settings)
        want, _ = _plain(logits, uniform, **settings)
        assert torch.equal(got.tokens, want), (k, p)
        _exact_check(logits, uniform, settings, got.tokens, got.log_prob)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [131072, 262144])
def test_many_long_rows_of_near_equal_logits(dtype, vocab):
    """Enough rows for one block each: a bin of its sums holds up to the whole
    row, 2^18 masses of 2^35."""
    from mamba4_b200 import sample_tokens

    rows = 150
    g = torch.Generator(device="cuda").manual_seed(vocab)
    spread = torch.tensor([0.0, 1e-3, 0.1, 0.3, 1.0], device="cuda")[torch.arange(rows, device="cuda") % 5]
    logits = (spread[:, None] * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    logits[75:, 1::4] -= 3.0
    uniform = torch.rand(rows, generator=g, device="cuda")
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.arange(rows, device="cuda") // 5 % len(v)]  # noqa: E731
    settings = dict(temperature=torch.ones(rows, device="cuda"), top_k=pick(0, vocab - 9, 70000).to(torch.int32),
                    top_p=pick(0.9, 0.5, 0.999, 1.0), min_p=torch.zeros(rows, device="cuda"))
    got = sample_tokens(logits, uniform, **settings)
    for r in range(0, rows, 50):
        part = {n: v[r:r + 50] for n, v in settings.items()}
        want, _ = _plain(logits[r:r + 50], uniform[r:r + 50], **part)
        assert torch.equal(got.tokens[r:r + 50], want), r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_different_logits_of_one_rank_value(dtype, rows):
    """z = (max - x) / T rounds different logits together: they rank by index
    then, and a row draws the same token whatever rows are beside it."""
    from mamba4_b200 import sample_tokens

    g = torch.Generator().manual_seed(12)
    tiny = 1e-30 * (1 + torch.randperm(1000, generator=g)).float()
    crowd = torch.cat((torch.tensor([1.0]), tiny))[torch.randperm(1001, generator=g)]
    pair = torch.full((1001,), -100.0)
    pair[0], pair[8], pair[16] = 1.0, 1.0 + 2.0 ** -23, 100.0
    near = 1e-10 * tiny / 1e-30
    for logits, temperature in ((crowd, 1.0), (crowd, 0.3), (pair, 10.0), (near, 3e38), (tiny * 1e-12, 4.0)):
        logits = logits.to(dtype).cuda()[None].repeat(rows, 1)
        for top_k in (1, 2, 5, 50, 127):
            for u in (0.0, 0.4, 0.9999):
                settings = dict(temperature=torch.full((rows,), temperature, device="cuda"),
                                top_k=torch.full((rows,), top_k, dtype=torch.int32, device="cuda"),
                                top_p=torch.ones(rows, device="cuda"), min_p=torch.zeros(rows, device="cuda"))
                uniform = torch.full((rows,), u, device="cuda")
                got = sample_tokens(logits, uniform, **settings)
                want, _ = _plain(logits, uniform, **settings)
                assert torch.equal(got.tokens, want), (temperature, top_k, u)


def test_whole_numbers_as_settings():
    """Per-row settings of any number type: only top_k is a count."""
    from mamba4_b200 import sample_tokens

    logits, uniform = 1e6 * torch.randn(4, 50, device="cuda"), torch.rand(4, device="cuda")
    want = sample_tokens(logits, uniform, temperature=torch.full((4,), 1e6, device="cuda"))
    got = sample_tokens(logits, uniform, temperature=torch.full((4,), 10 ** 6, device="cuda"))
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.log_prob, want.log_prob)
    want = sample_tokens(logits, uniform, top_k=3)
    for k in (torch.full((4,), 3.0, device="cuda"), torch.full((4,), 3, dtype=torch.uint8, device="cuda")):
        assert torch.equal(sample_tokens(logits, uniform, top_k=k).tokens, want.tokens)


def test_several_host_threads():
    """One row each (16 blocks: a size asked of the driver once), from threads that start together."""
    import threading

    from mamba4_b200 import sample_tokens

    logits, uniform = torch.randn(8, 60000, device="cuda"), torch.rand(8, device="cuda")
    got, start = [None] * 8, threading.Barrier(8)

    def run(i):
        start.wait()
        got[i] = sample_tokens(logits[i:i + 1], uniform[i:i + 1], top_p=0.9).tokens

    threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(8):
        assert torch.equal(got[i], sample_tokens(logits[i:i + 1], uniform[i:i + 1], top_p=0.9).tokens)
