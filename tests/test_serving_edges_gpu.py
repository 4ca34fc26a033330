"""The serving operators at the edges of what they take, on the GPU.  Tolerances as in
test_paged_gpu.py and test_logprobs_gpu.py."""
import math

import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib
from test_logprobs_gpu import rows
from test_paged_gpu import check, check_attention, check_step, make, ref_attention, run_attention, run_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", range(4, 128, 8))
@pytest.mark.parametrize("Hq", [2, 16])
def test_dense_rows_on_8_byte_boundaries(cuda_device, D, Hq):
    """Pages of dense rows of every odd multiple of 4, used up to the pool's last row; the
    values that follow a row in memory are the next one's."""
    s = make(cuda_device, [96, 31, 160], Hq, 2, D, 32, seed=D, spare=0, room=0)
    assert s["kp"].is_contiguous() and s["table"].max() == s["kp"].shape[0] - 1
    check_step(s, *run_step(s, append=False))
    check_attention(s, run_attention(s))
    _lib.check_status()


@pytest.mark.parametrize("gq", [1, 16])
def test_weights_keep_the_bits_of_fp32(cuda_device, gq):
    """Sums that cancel: two tokens of score 0 hold p b as two bf16 parts, against one of
    weight p = exp(-t / 32) and value b, so what is left shows p's last bits.  The score is exact
    but for log2 e's rounding and its own, 2^-23 for |z| < 1; exp2 adds 2^-22, and at most six fp32
    sums on the way half a step of the sum of |p x| or, truncated, a whole one: 9 2^-23 in all,
    12 allowed.  A weight of 16 bits is off by up to 2^-18, 32 2^-23."""
    H, D = 32, 64
    s = make(cuda_device, [3], H * gq, H, D, 16, seed=5)
    s["scale"] = 1 / 32
    t = torch.linspace(1, 22, H, device=cuda_device).bfloat16().double()
    p = torch.exp(-t / 32)[:, None]
    page = int(s["table"][0, 0])
    b = s["xp"][page, :, 1].double()
    s["kp"][page, :, :3] = 0
    s["kp"][page, :, 1, 0] = -t.bfloat16()
    high = (p * b).bfloat16()
    s["xp"][page, :, 0], s["xp"][page, :, 2] = -high, -(p * b - high.double()).bfloat16()
    s["q"].zero_()
    s["q"][..., 0] = 1
    s["k"].zero_()                                   # the step's own token: weight 1, value v
    s["v"].zero_()                                   # less e^-32 of the others, next to nothing
    ref, mag, _ = ref_attention(s, 0)
    assert (ref.abs() < 2.0 ** -16 * mag).all()
    check(run_attention(s)[0, 0], ref, 12 * 2.0 ** -23 * mag)
    o, xn = run_step(s, append=False)
    ref, mag, _ = ref_attention(s, 0, (s["k"][0], xn[0]))
    check(o[0, 0], ref, 12 * 2.0 ** -23 * mag)
    _lib.check_status()


def test_a_captured_batch_step_follows_the_bookkeeping(cuda_device):
    """reserve, replay, advance, with forks, frees, moved pages and another batch's steps in
    between: the same bits as a twin cache's eager steps, and no page but the reserved rows
    changes."""
    H, D, ps = 2, 68, 16
    g = torch.Generator(device=cuda_device).manual_seed(9)
    rn = lambda *shape: torch.randn(*shape, generator=g, device=cuda_device).bfloat16()
    caches = [lb.PagedCache(2, H, D, 60, ps, device=cuda_device) for _ in range(2)]
    batches = [c.batch(c.new(3)) for c in caches]
    prompt = [rn(3, H, 40, D) for _ in range(2)]
    for c, b in zip(caches, batches):
        c.key_pages.zero_()
        c.x_pages.zero_()
        b.reserve([40, 15, 31])
        for layer in range(2):
            b.append(layer, *prompt)
        b.advance()
    q, k, v = rn(3, 4, 1, D), rn(3, H, 1, D), rn(3, H, 1, D)
    scale = D ** -0.5
    batches[0].reserve(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [batches[0].step(layer, q, k, v, scale) for layer in range(2)]
    for step in range(40):
        for t in (q, k, v):
            t.copy_(rn(*t.shape))
        for c, b in zip(caches, batches):
            if step == 3:
                c.fork(b.sequences[1])
            if step == 9:
                c.free(3)
            if step == 12:
                spare = c.batch(c.new(2))
                spare.reserve(30)
                for layer in range(2):
                    spare.append(layer, prompt[0][:2], prompt[1][:2])
                spare.advance()
            if step == 20:
                c.free(4)
                c.compact()
            b.reserve(1)
        graph.replay()
        batches[0].advance()
        want = [batches[1].step(layer, q, k, v, scale) for layer in range(2)]
        batches[1].advance()
        for (o, x), (o2, x2) in zip(out, want):
            assert torch.equal(o, o2) and torch.equal(x, x2)
        for t in ("key_pages", "x_pages"):
            assert torch.equal(getattr(caches[0], t), getattr(caches[1], t)), step
    assert batches[0].lengths.tolist() == batches[0].host_lengths == [80, 55, 71]
    _lib.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_gradient_of_tokens_outside_the_vocabulary(cuda_device, dtype):
    """NaN like their log probability, whichever side they are on; without a factor for it, and
    for -100, the entropy's alone."""
    x = torch.randn(8, 50, generator=torch.Generator(device=cuda_device).manual_seed(1), device=cuda_device).to(dtype)
    t = torch.tensor([1, 50, -1, 2 ** 40, -99, -100, 60, -7], device=cuda_device)
    gl = torch.tensor([1., 2., -1., .5, 3., 1., 0., 0.], device=cuda_device)
    for ge in (torch.zeros(8, device=cuda_device), torch.linspace(-1, 1, 8, device=cuda_device)):
        x.requires_grad_(True)
        got = lb.token_logprobs(x, t)
        with pytest.raises(_lib.LucidError, match="a token lies outside the vocabulary"):
            _lib.check_status()
        d, = torch.autograd.grad([got.logprobs, got.entropy], x, [gl, ge])
        assert d[1:5].isnan().all() and torch.isfinite(d[[0, 5, 6, 7]]).all()
        alone = lb.token_logprobs(x, None)
        want, = torch.autograd.grad(alone.entropy, x, ge)
        assert torch.equal(d[5:], want[5:])
    _lib.check_status()


def test_append_tells_a_page_from_a_length(cuda_device):
    """One cause each: a page missing inside the table, rows past a table of valid pages."""
    for table, count, match in (([0, -1, 2], 20, "a page of the block table"), ([0, 9, 2], 20, "a page of the block table"),
                                ([0, 1, 2], 49, "past the block table")):
        kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device)
        xp = torch.zeros_like(kp)
        k = torch.ones(1, 2, 60, 64, dtype=torch.bfloat16, device=cuda_device)
        n, c = (torch.tensor([v], dtype=torch.int32, device=cuda_device) for v in (0, count))
        lb.paged_append(k, k, kp, xp, torch.tensor([table], dtype=torch.int32, device=cuda_device), n, c)
        with pytest.raises(_lib.LucidError, match=match):
            _lib.check_status()
        written = [0, 1, 2] if count == 49 else [0]
        assert torch.equal(kp, xp) and [p for p in range(4) if kp[p].any()] == written and (kp[written] == 1).all()
    _lib.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,V", [(3, 5), (4, 1000), (2, 32001)])
def test_the_gradient_of_the_entropy_without_tokens(cuda_device, dtype, R, V):
    """Tolerance of the gradient as in test_logprobs_gpu.py, g_lp 0."""
    x = rows(cuda_device, (R, V), dtype, seed=V)
    x[0, V // 2] = -math.inf
    x.requires_grad_(True)
    ge = torch.randn(R, generator=torch.Generator(device=cuda_device).manual_seed(3), device=cuda_device)
    got = lb.token_logprobs(x, None)
    assert got.logprobs is None
    d, = torch.autograd.grad(got.entropy, x, ge)
    lp = torch.log_softmax(x.detach().double(), -1)
    p, lpf = lp.exp(), torch.where(lp > -math.inf, lp, 0.0)
    h = -(p * lpf).sum(-1, keepdim=True)
    want = -ge[:, None] * p * (lpf + h)
    mag = ge.abs()[:, None] * (lpf.abs() + h + 1) * p
    tol = torch.finfo(dtype).eps / 2 * want.abs() + mag * (V / 512 + 28 + 2 * lpf.abs()) * 2.0 ** -23 * (1 + math.log(V)) \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert d.dtype == dtype and ((d.double() - want).abs() <= tol).all()
    _lib.check_status()


def test_forward_mode_is_refused_on_the_gpu(cuda_device):
    from torch.autograd import forward_ad
    x = torch.randn(2, 5, device=cuda_device)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        lb.token_logprobs(forward_ad.make_dual(x, x), None)


@pytest.mark.parametrize("gq", [1, 9])
def test_long_sums_are_rounded_not_cut(cuda_device, gq):
    """A long sequence's first half holds N values b with weight p = exp(-t / 32), with a token
    of score 0 and value 0 in every 16, so that every warp weighs by the same maximum; the
    second half's tokens have score 0, values that take N p b away again and few bits, so
    their sums are exact.  Every CTA adds up about 128 tiles a row.  What is left, relative to the
    sum of |p x|, of which the first half is one half, in units of 2^-23:
      p: exp2 2, its argument 1; a tile's own products and sums, cut at three places, 3; so 3 in all
      sums rounded to nearest: each at most half a unit of the sum so far, 128 of them 32, so
      16 in all, without direction: next to nothing in the mean over heads and columns
    Sums cut off at fp32's last digit, at 384 places, left 15 in the mean and up to 105."""
    H, D, ps, n = 32, 16, 64, 128 * 444 // 32 * 64
    kp = torch.zeros(n // ps, H, ps, D, dtype=torch.bfloat16, device=cuda_device)
    xp = torch.zeros_like(kp)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    t = torch.linspace(1, 22, H, device=cuda_device).bfloat16().double()[:, None]
    b = (1 + torch.rand(H, D, generator=g, device=cuda_device)).bfloat16().double()
    half = n // ps // 2
    held = torch.arange(ps, device=cuda_device) % 16 != 0
    kp[:half, :, held, 0] = -t.bfloat16()
    xp[:half, :, held] = b.bfloat16()[:, None]
    total = half * int(held.sum()) * torch.exp(-t / 32) * b
    second = half * ps - 3
    rest, each = total.clone(), (total / second).bfloat16()
    xp[half:] = -each[:, None]
    rest -= second * each.double()
    for i in range(3):                               # the last three tokens take the rest
        part = rest.bfloat16()
        xp[-1, :, ps - 1 - i] = -part
        rest -= part.double()
    assert (rest.abs() < 2.0 ** -24 * total).all()
    weight = half * int(held.sum()) * torch.exp(-t / 32) + half * 4 + half * ps
    q = torch.zeros(1, H * gq, 1, D, dtype=torch.bfloat16, device=cuda_device)
    q[..., 0] = 1
    table = torch.arange(n // ps, dtype=torch.int32, device=cuda_device)[None]
    o = lb.paged_decode_attention(q, kp, xp, table, torch.tensor([n], dtype=torch.int32, device=cuda_device), 1 / 32)
    off = (o.view(H, gq, D).double() - (rest / weight)[:, None]) * weight[:, None] / (2 * total)[:, None] * 2.0 ** 23
    assert off.abs().max() <= 3 + 16 + 1 and off.mean().abs() <= 3 + 1, (off.abs().max(), off.mean())
    _lib.check_status()
