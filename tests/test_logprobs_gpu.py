"""Token log probabilities, entropies, alternatives and their gradient against 64 bits.

Tolerances.  A row's sum is V / 512 terms in turn in a thread, then a tree: with n =
V / 512 + 24 roundings and exp2's 2 ulp, l and w are within n 2^-23 of themselves, so
    |logprob - ref| <= n 2^-23 + |ref| 2^-22            (the log, the difference)
    |entropy - ref| <= 2 n 2^-23 (1 + ln V)             (log2 l and w / l are at most ln V)
Where many rows get a warp each, a thread adds V / 64 terms of half a step, n = V / 128 + 24.
p is within (n + 2 |log p| + 4) 2^-23 of itself; the gradient adds half a step of its type
(finfo.eps / 2, or half the smallest subnormal)."""
import math

import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def slack(V, wide=512):
    return (V / wide + 24) * 2.0 ** -23


def reference(x, tokens):
    assert int(tokens.max()) < x.shape[-1]                       # torch's gather would assert on the device
    lp = torch.log_softmax(x.double(), -1)
    h = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(-1)
    chosen = torch.where(tokens >= 0, lp.gather(-1, tokens.clamp(min=0)[..., None])[..., 0], 0.0)
    return lp, chosen, h


def ranked(x, k):
    """The k largest of each row, ties to the lowest index: a stable sort."""
    return torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[..., :k]


def check(x, tokens, top, wide=512):
    V = x.shape[-1]
    err = slack(V, wide)
    got = lb.token_logprobs(x, tokens, top=top)
    lp, chosen, h = reference(x, tokens)
    assert got.logprobs.shape == got.entropy.shape == x.shape[:-1] and got.top_tokens.shape == (*x.shape[:-1], top)
    live = (x == x).all(-1) & ~(x == math.inf).any(-1) & (x > -math.inf).any(-1)     # else without a distribution
    assert got.entropy[~live].isnan().all() and got.top_logprobs[~live].isnan().all() and (got.top_tokens[~live] == -1).all()
    assert (got.logprobs[~live].isnan() == (tokens[~live] >= 0)).all()
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == F32 and got.top_tokens.dtype == torch.int64
    whole, got = got, lb.TokenLogprobs(*(part[live] for part in got))
    x, lp, chosen, h = x[live], lp[live], chosen[live], h[live]
    inf = chosen < -torch.finfo(F32).max                         # -6e38 has no fp32 value but -inf
    assert (got.logprobs[inf] == -math.inf).all()
    assert ((got.logprobs - chosen).abs()[~inf] <= err + chosen.abs()[~inf] * 2.0 ** -22).all(), (got.logprobs - chosen).abs().max()
    assert ((got.entropy - h).abs() <= 2 * err * (1 + math.log(V))).all(), (got.entropy - h).abs().max()
    if top:
        want = ranked(x, top)
        assert torch.equal(got.top_tokens, want)
        ref = lp.gather(-1, want)
        fin = ref >= -torch.finfo(F32).max
        assert ((got.top_logprobs - ref).abs()[fin] <= err + ref.abs()[fin] * 2.0 ** -22).all()
        assert (got.top_logprobs[~fin] == -math.inf).all()
    _lib.check_status()
    return whole


def rows(dev, shape, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (spread * torch.randn(*shape, generator=g, device=dev)).to(dtype)


def some_tokens(x, seed=0):
    t = torch.randint(0, x.shape[-1], x.shape[:-1], generator=torch.Generator().manual_seed(seed)).to(x.device)
    if t.numel() > 2:
        t.view(-1)[1] = -100
    return t


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (3, 2, 2), (5, 7, 0), (4, 100, 64), (3, 511, 5), (3, 513, 20), (2, 4097, 64),
                                     (5, 32000, 20), (2, 50021, 1), (1, 200003, 50), (300, 1000, 3)])
def test_matches_64_bits(cuda_device, dtype, R, V, top):
    x = rows(cuda_device, (R, V), dtype, seed=V)
    check(x, some_tokens(x), top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("R,V,top", [(1000, 9001, 20), (950, 20000, 24), (950, 8192, 25), (3, 174683, 50), (901, 4097, 0)])
def test_many_rows_and_long_rows(cuda_device, dtype, R, V, top):
    """Both block widths over several batches of a row, the second one's alternatives listed
    by the first one's threshold."""
    x = rows(cuda_device, (R, V), dtype, seed=R)
    check(x, some_tokens(x), top)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("R,V,top", [(3000, 9001, 20), (3557, 31000, 24), (7111, 2049, 1), (3000, 40, 24), (3000, 185, 24),
                                     (3001, 32768, 5), (3001, 5, 5), (300, 2560, 24), (1300, 50000, 24),
                                     (2000, 130000, 20)])
def test_a_warp_a_row(cuda_device, dtype, R, V, top):
    """Many rows with few alternatives; as many rows as warps, and some more."""
    x = rows(cuda_device, (R, V), dtype, seed=R)
    check(x, some_tokens(x), top, wide=128)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_a_warp_a_row_of_any_kind(cuda_device, dtype):
    R, V = 3001, 12003
    low = torch.finfo(dtype).min
    x = rows(cuda_device, (R, V), dtype, seed=8)
    x[0] = 0                                                     # all equal
    x[1, 8000:] = 30                                             # thousands best
    x[2, 7::50] = 30
    x[3, :], x[3, 100:103] = 1, 3                                # three above many ties
    x[4] = x[4].float().round().to(dtype)
    x[5, ::2], x[5, 1::2] = -0.0, 0.0
    x[6] = torch.sort(x[6]).values
    x[7] = torch.sort(-x[7].abs(), descending=True).values       # keys of negative numbers
    x[8] = torch.sort(x[8]).values.view(3, V // 3).t().reshape(-1)
    x[9, : V // 2] = -math.inf                                   # a start that says nothing
    x[10, : V - 40] = low
    x[11, 1:] = -math.inf                                        # one left, three left, fewer than asked for
    x[12, :], x[12, [5, 2000, 12002]] = low, torch.tensor([1.0, 2.0, 1.0], dtype=dtype, device=cuda_device)
    x[13, 3:] = low
    x[14, ::1700] = 50                                           # next to each other in no lane
    x[15] = low
    x[16], x[16, 256 * 8:256 * 9] = -40, x[17, 256 * 8:256 * 9]  # all of the large ones in a few vectors
    t = some_tokens(x)
    t[11] = 0
    check(x, t, 20, wide=128)
    check(x[:, 1:-1], t.clamp(max=V - 3), 24, wide=128)          # odd row starts
    broken = x.clone()
    broken[20], broken[21, 17], broken[22, V - 1], broken[3000, 600] = -math.inf, math.nan, math.inf, math.nan
    got = lb.token_logprobs(broken, t, top=20)
    bad = [20, 21, 22, 3000]
    assert got.entropy[bad].isnan().all() and got.logprobs[bad].isnan().all()
    assert got.top_logprobs[bad].isnan().all() and (got.top_tokens[bad] == -1).all()
    keep = torch.ones(R, dtype=torch.bool, device=cuda_device)
    keep[bad] = False
    same = lb.token_logprobs(x, t, top=20)
    for a, b in zip(got, same):
        assert torch.equal(a[keep], b[keep])                     # the others do not notice, bit for bit


def test_a_warp_a_row_with_its_gradient(cuda_device):
    """The row statistics that the gradient needs, next to alternatives, in strided rows."""
    x = rows(cuda_device, (2, 1502, 3001), F32, seed=5).requires_grad_(True)
    t = some_tokens(x[:, :-1])
    got = lb.token_logprobs(x[:, :-1], t, top=4)
    gl, ge = rows(cuda_device, got.entropy.shape, F32, seed=6), rows(cuda_device, got.entropy.shape, F32, seed=7)
    d, = torch.autograd.grad((got.logprobs, got.entropy), x, (gl, ge))
    lp, _, h = reference(x.detach()[:, :-1], t)
    p, real = lp.exp(), (t >= 0)[..., None]
    one = torch.zeros_like(p).scatter_(-1, t.clamp(min=0)[..., None], 1.0) * real
    gl, ge = gl.double()[..., None] * real, ge.double()[..., None]
    want = gl * (one - p) - ge * p * (lp + h[..., None])
    mag = (gl.abs() + ge.abs() * (lp.abs() + h[..., None] + 1)) * p     # as in test_gradient_matches_formula, V / 128 terms
    tol = 2.0 ** -24 * want.abs() + mag * (3001 / 128 + 28 + 2 * lp.abs()) * 2.0 ** -23 * (1 + math.log(3001)) \
        + gl.abs() * one * 2.0 ** -23 + torch.finfo(F32).smallest_normal
    assert not d[:, -1].any()
    assert ((d[:, :-1] - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V,top", [(905, 20000, 20), (2, 120000, 50)])
def test_a_first_batch_that_says_nothing(cuda_device, dtype, R, V, top):
    """The start of a row far below the rest, or banned: the candidate list overflows and is
    made again by the final threshold, or, in constant rows, left for a scan."""
    x = rows(cuda_device, (R, V), dtype, seed=V)
    x[:, : V // 2] -= 40
    x[0, : V // 2] = -math.inf
    x[1] = 1.0
    check(x, some_tokens(x), top)
    x[0], x[0, :7] = -math.inf, 0.5
    x[1, V // 2:] = 2.0
    check(x, torch.zeros(R, dtype=torch.int64, device=cuda_device), top)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_are_read_in_place(cuda_device, dtype):
    x = rows(cuda_device, (3, 6, 1003), dtype)
    check(x[:, :-1], some_tokens(x[:, :-1]), 5)                  # odd row starts, a gap between the outer rows
    check(x[:, 2], some_tokens(x[:, 2]), 5)
    check(x[..., 1:-1], some_tokens(x[..., 1:-1]), 5)
    check(x.transpose(0, 1), some_tokens(x.transpose(0, 1)), 5)
    check(x[:1].expand(3, 6, 1003), some_tokens(x), 2)
    check(x[..., ::2], some_tokens(x[..., ::2]), 2)                        # strided vocabulary: copied
    check(x.reshape(3, 2, 3, 1003)[:, :, 1:].transpose(0, 2), some_tokens(x.reshape(3, 2, 3, 1003)[:, :, 1:].transpose(0, 2)), 2)
    check(x[1, 1], torch.tensor(4, device=cuda_device), 2)       # a single row
    check(x, some_tokens(x).int(), 0)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_ties_go_to_the_lowest_index(cuda_device, dtype):
    V = 5000
    x = torch.zeros(6, V, dtype=dtype, device=cuda_device)       # all equal: more ties than the list holds
    x[1, 4000:] = 1                                              # a thousand best
    x[2, 7::50] = 2
    x[3, 100:103] = 3                                            # three above many ties
    x[4] = (rows(cuda_device, (V,), F32).round()).to(dtype)
    x[5, ::2] = -0.0
    check(x, some_tokens(x), 20)
    check(x, some_tokens(x), 64)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rising", [False, True])
def test_sorted_rows(cuda_device, dtype, rising):
    """Everything large side by side: thread maxima say little, the threshold is made
    exact by histograms (fp32) or the ties are scanned (bf16)."""
    x = torch.sort(rows(cuda_device, (3, 32000), dtype, seed=9), -1, descending=not rising).values
    x[1] = -x[1].abs()                                           # keys of negative numbers
    check(x, some_tokens(x), 64)
    check(x, some_tokens(x), 20)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_banned_entries(cuda_device, dtype):
    V = 3001
    for low in (-math.inf, torch.finfo(dtype).min):
        x = rows(cuda_device, (6, V), dtype, seed=1)
        x[0, 1:] = low                                           # one token left
        x[1, :] = low
        x[1, [5, 2000, 2999]] = torch.tensor([1.0, 2.0, 1.0], dtype=dtype, device=cuda_device)
        x[2, torch.rand(V, device=cuda_device) < 0.95] = low
        x[3, :1500] = low
        x[4, 3:] = low                                           # fewer left than asked for
        t = torch.tensor([0, 5, -100, 2000, 17, 9], device=cuda_device)
        check(x, t, 10)
    x[:] = torch.finfo(dtype).min                                # a mask of the lowest value alone: uniform
    got = check(x, t, 10)
    assert (got.entropy - math.log(V)).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_rows_without_a_distribution(cuda_device, dtype):
    x = rows(cuda_device, (5, 900), dtype)
    x[0] = -math.inf
    x[1, 17] = math.nan
    x[2, 899] = math.inf
    x[3, 3] = -math.inf
    t = torch.tensor([1, 2, -100, 3, 4], device=cuda_device)
    x.requires_grad_(True)
    got = lb.token_logprobs(x, t, top=3)
    assert got.entropy[:3].isnan().all() and got.logprobs[:2].isnan().all() and got.logprobs[2] == 0
    assert got.top_logprobs[:3].isnan().all() and (got.top_tokens[:3] == -1).all()
    assert got.logprobs[3] == -math.inf and torch.isfinite(got.entropy[3:]).all() and torch.isfinite(got.top_logprobs[3:]).all()
    # no gradient is asked of the broken rows: none comes out; else it is NaN
    g = torch.tensor([0.0, 0.0, 1.0, 1.0, 1.0], device=cuda_device)
    d, = torch.autograd.grad(got.logprobs, x, g, retain_graph=True)
    assert not d[:3].any() and torch.isfinite(d).all()
    d, = torch.autograd.grad(got.entropy, x, torch.ones(5, device=cuda_device))
    assert d[:3].isnan().all() and torch.isfinite(d[3:]).all()


def test_extreme_values(cuda_device):
    """Rows far from zero lose no digits; values next to fp32's ends do not overflow."""
    x = rows(cuda_device, (4, 1000), F32, seed=2) + torch.tensor([[1e4], [-1e4], [0.0], [0.0]], device=cuda_device)
    x[2, 0] = 3e38
    x[3] = -3e38
    x[3, 1] = 3e38
    check(x, some_tokens(x), 8)


def test_tokens_outside_the_vocabulary(cuda_device):
    x = rows(cuda_device, (4, 50), F32)
    for bad in (50, -1, 2 ** 40, -99):
        t = torch.tensor([1, bad, 2, 3], device=cuda_device)
        got = lb.token_logprobs(x, t)
        with pytest.raises(_lib.LucidError, match="a token lies outside the vocabulary"):
            _lib.check_status()
        assert got.logprobs[1].isnan() and torch.isfinite(got.logprobs[[0, 2, 3]]).all()
    _lib.check_status()


def test_refusals_and_empty(cuda_device):
    x = rows(cuda_device, (4, 50), F32)
    t = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    for call, err in ((lambda: lb.token_logprobs(x.double(), t), TypeError), (lambda: lb.token_logprobs(x, t.float()), TypeError),
                      (lambda: lb.token_logprobs(x, t[:3]), ValueError), (lambda: lb.token_logprobs(x, t.cpu()), ValueError),
                      (lambda: lb.token_logprobs(x, t, top=51), ValueError), (lambda: lb.token_logprobs(x, t, top=-1), ValueError),
                      (lambda: lb.token_logprobs(rows(cuda_device, (2, 99), F32), None, top=65), ValueError),
                      (lambda: lb.token_logprobs(x[:, :0], t), ValueError), (lambda: lb.token_logprobs(x[0, 0], None), ValueError)):
        with pytest.raises(err):
            call()
    got = lb.token_logprobs(x[:0], t[:0], top=3)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 3)
    got = lb.token_logprobs(x, None, top=2)
    assert got.logprobs is None and torch.equal(got.top_tokens, ranked(x, 2))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("R,V", [(3, 5), (4, 1000), (3, 32001), (2, 70000)])
def test_gradient_matches_formula(cuda_device, dtype, R, V):
    x = rows(cuda_device, (R, V + 3), dtype, seed=V)[:, 1:V + 1].requires_grad_(True)   # rows off the vector grid
    t = some_tokens(x)
    with torch.no_grad():
        x[0, V // 2] = -math.inf
        t[0] = 0
    g = torch.Generator(device=cuda_device).manual_seed(3)
    gl, ge = (torch.randn(R, generator=g, device=cuda_device) for _ in range(2))
    lp, _, h = reference(x.detach(), t)
    p = lp.exp()
    lpf = torch.where(p > 0, lp, 0.0)
    one = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0) * (t >= 0)[:, None]
    d_lp = (t >= 0)[:, None] * gl[:, None] * (one - p)
    d_h = -ge[:, None] * p * (lpf + h[:, None])
    got = lb.token_logprobs(x, t, top=1)
    assert got.logprobs.requires_grad and got.entropy.requires_grad and not got.top_logprobs.requires_grad
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    for outs, grads, want in (([got.logprobs], [gl], d_lp), ([got.entropy], [ge], d_h),
                              ([got.logprobs, got.entropy], [gl, ge], d_lp + d_h)):
        d, = torch.autograd.grad(outs, [x], grads, retain_graph=True)
        mag = (gl.abs()[:, None] + ge.abs()[:, None] * (lpf.abs() + h[:, None] + 1)) * p
        tol = torch.finfo(dtype).eps / 2 * want.abs() + mag * (V / 512 + 28 + 2 * lpf.abs()) * 2.0 ** -23 * (1 + math.log(V)) \
            + gl.abs()[:, None] * one * 2.0 ** -23 + tiny
        assert d.dtype == dtype and d.shape == x.shape
        assert ((d.double() - want).abs() <= tol).all(), ((d.double() - want).abs() - tol).max()


def test_gradient_matches_differences(cuda_device):
    """Central differences of f = sum gl logprob + ge entropy along random directions, h =
    2^-6: truncation below h^2 |f'''| / 6 with third derivatives of order |d|^3, noise below
    40 values' roundings (2^-20 each) over 2 h."""
    R, V, h = 4, 41, 2.0 ** -6
    x = rows(cuda_device, (R, V), F32, seed=4, spread=1.0).requires_grad_(True)
    t = torch.tensor([3, 40, 0, 7], device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    gl, ge = (torch.randn(R, generator=g, device=cuda_device).double() for _ in range(2))

    def f(y):
        got = lb.token_logprobs(y, t)
        return (gl * got.logprobs.double() + ge * got.entropy.double()).sum()
    d, = torch.autograd.grad(f(x), x)
    for _ in range(6):
        u = torch.randn(R, V, generator=g, device=cuda_device)
        u /= u.norm()
        with torch.no_grad():
            diff = (f(x + h * u) - f(x - h * u)) / (2 * h)
        assert abs(diff - (d.double() * u).sum()) <= h * h * float(gl.abs().sum() + 5 * ge.abs().sum()) + 40 * 2.0 ** -20 / (2 * h)


def test_gradient_through_views_and_sums(cuda_device):
    """A broadcast leaf, a slice of a wider tensor, only one of the outputs used, a summed
    loss: the gradients add up as torch's own do."""
    base = rows(cuda_device, (4, 600), F32, seed=6)
    t = some_tokens(base.expand(3, 4, 600))
    for view in (lambda a: a.expand(3, 4, 600), lambda a: a[:, 100:500], lambda a: a.t().contiguous().t()[1:]):
        a, b = (base.clone().requires_grad_(True) for _ in range(2))
        va, vb = view(a), view(b)
        tt = t[tuple(slice(0, n) for n in va.shape[:-1])] if va.dim() == 3 else t[0, :va.shape[0]].clamp(max=va.shape[-1] - 1)
        (lb.token_logprobs(va, tt).logprobs.sum() * 2).backward()
        lp = torch.log_softmax(vb.double(), -1)
        (torch.where(tt >= 0, lp.gather(-1, tt.clamp(min=0)[..., None])[..., 0], 0.0).sum() * 2).backward()
        assert (a.grad - b.grad).abs().max() < 1e-5
    got = lb.token_logprobs(a, t[0])
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(got.entropy.sum(), a, create_graph=True)
        d.sum().backward()


def test_captured_forward_and_backward(cuda_device):
    """Captured with torch.autograd.grad, replayed on new logits while an eager graph of the
    same leaf is alive."""
    x = rows(cuda_device, (16, 999), BF, seed=7).requires_grad_(True)
    t = some_tokens(x)
    ones = torch.ones(16, device=cuda_device)

    def both():
        got = lb.token_logprobs(x, t, top=4)
        d, = torch.autograd.grad([got.logprobs, got.entropy], [x], [ones, ones])
        return got.logprobs, got.entropy, got.top_tokens, d
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    alive = lb.token_logprobs(x, t)
    for seed in (8, 9):
        with torch.no_grad():
            x.data.copy_(rows(cuda_device, (16, 999), BF, seed=seed))
        g.replay()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert alive.logprobs.requires_grad


def test_two_runs_and_two_streams_agree(cuda_device):
    x = rows(cuda_device, (64, 32000), BF, seed=10)
    t = some_tokens(x)
    want = lb.token_logprobs(x, t, top=20)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(lb.token_logprobs(x, t, top=20))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))
