"""Paged decoding, appends and page copies on the GPU against plain 64-bit formulas.

Tolerances.  q k^T is a sum of exact products in fp32: with A the largest sum of |q k| s
over a row's tokens, a score is off by at most (D/16 + 5) 2^-23 A, and a weight by twice that
relative to itself (its numerator and the denominator), plus 2^-15 for the two-part bf16
weight (half a step of the second part: 2^-8 2^-8), exp2 and the fp32 sums.  The output
adds half a bf16 step, 2^-8 of its value:
    |o - ref|     <= 2^-8 |ref| + (2^-15 + 2 (D/16 + 5) 2^-23 A) sum p |x|
In the update the exponent, up to 16 in log2 units, also carries the two reciprocal roots
(2 ulp each) and its own roundings, below 8 2^-23 16 = 2^-16, and e is not normalised:
    |x_new - ref| <= 2^-8 |ref| + (2^-14 + (D/16 + 5) 2^-23 16) sum e |x|
(the largest |k^.k^| s log2 e is s D log2 e <= 16.4 at D = 128)."""
import numpy as np
import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib

pytestmark = pytest.mark.gpu


def make(dev, lens, Hq, Hkv, D, ps, seed=0, spare=2, pad=0, poison=True, room=1):
    """A batch over a shuffled pool.  Rows that no sequence owns hold NaN.  pad: extra
    elements between the rows of the pools (4: rows on 8-byte boundaries only)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    need = [max(0, -(-(max(n, 0) + room) // ps)) for n in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    full = [torch.full((P, Hkv, ps, D + pad), float("nan"), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    kp, xp = (f[..., :D] for f in full)
    lean = rn(Hkv, 1, D)
    for b, n in enumerate(lens):
        for t0 in range(0, max(n, 0), ps):
            r = min(ps, n - t0)
            p = int(table[b, t0 // ps])
            kp[p, :, :r] = (0.8 * rn(Hkv, r, D) + 0.6 * lean).bfloat16()
            xp[p, :, :r] = rn(Hkv, r, D).bfloat16()
    B = len(lens)
    s = dict(q=rn(B, Hq, 1, D).bfloat16(), k=(0.8 * rn(B, Hkv, 1, D) + 0.6 * lean).bfloat16(), v=rn(B, Hkv, 1, D).bfloat16(),
             kp=kp, xp=xp, table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev), scale=D ** -0.5)
    return s


def rows_of(s, b):
    """Sequence b's cached keys and solved values, [Hkv, n, D] in 64 bits."""
    n, ps = max(int(s["lens"][b]), 0), s["kp"].shape[2]
    ids = s["table"][b].long()[torch.arange(n, device=s["kp"].device) // ps]
    at = torch.arange(n, device=s["kp"].device) % ps
    return (s["kp"][ids, :, at].double().transpose(0, 1), s["xp"][ids, :, at].double().transpose(0, 1))


def ref_update(s, b, eps=1e-5):
    """(x_new, sum e |x|) of sequence b."""
    k, x = rows_of(s, b)
    unit = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
    kn = s["k"][b].double()
    e = torch.exp(s["scale"] * unit(kn) @ unit(k).mT - 1.0 / s["scale"])
    return s["v"][b].double() - e @ x, e @ x.abs()


def ref_attention(s, b, new=None):
    """(o, sum p |x|, A) of sequence b; new: (key, solved value) of the new token."""
    k, x = rows_of(s, b)
    if new is not None:
        k, x = torch.cat([k, new[0].double()], 1), torch.cat([x, new[1].double()], 1)
    H, D = k.shape[0], k.shape[2]
    q = s["q"][b, :, 0].double().reshape(H, -1, D)
    if k.shape[1] == 0:
        z = torch.zeros_like(q).reshape(-1, D)
        return z, z, torch.zeros(z.shape[0], 1, device=z.device, dtype=z.dtype)
    p = torch.softmax(s["scale"] * q @ k.mT, -1)
    A = s["scale"] * (q.abs() @ k.abs().mT).amax(-1, keepdim=True)
    return (p @ x).reshape(-1, D), (p @ x.abs()).reshape(-1, D), A.reshape(-1, 1)


def check(got, ref, slack):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all() and (err <= 2.0 ** -8 * ref.abs() + slack).all(), \
        (err - 2.0 ** -8 * ref.abs() - slack).max().item()


def check_step(s, o, xn):
    D = s["kp"].shape[3]
    for b in range(len(s["lens"])):
        if int(s["lens"][b]) < 0:
            assert not o[b].any() and not xn[b].any()
            continue
        ref, mag = ref_update(s, b)
        check(xn[b], ref, (2.0 ** -14 + (D / 16 + 5) * 2.0 ** -23 * 16) * mag)
        ref, mag, A = ref_attention(s, b, (s["k"][b], xn[b]))
        check(o[b, 0], ref, (2.0 ** -15 + 2 * (D / 16 + 5) * 2.0 ** -23 * A) * mag)


def check_attention(s, o):
    D = s["kp"].shape[3]
    for b in range(len(s["lens"])):
        ref, mag, A = ref_attention(s, b)
        check(o[b, 0], ref, (2.0 ** -15 + 2 * (D / 16 + 5) * 2.0 ** -23 * A) * mag)


def run_step(s, **kw):
    return lb.paged_decode_step(s["q"], s["k"], s["v"], s["kp"], s["xp"], s["table"], s["lens"], s["scale"], 1e-5, **kw)


def run_attention(s):
    return lb.paged_decode_attention(s["q"], s["kp"], s["xp"], s["table"], s["lens"], s["scale"])


# lengths at every border of a 16-token warp slice, a 64-token tile and a page; head
# groups at the borders of the 8- and 16-row operands; every chunk width
CASES = [
    ([0], 4, 4, 128, 16), ([1], 4, 4, 128, 16), ([0, 1, 2], 8, 1, 68, 1),
    ([15, 16, 17, 31, 33], 8, 4, 64, 16), ([63, 64, 65, 127, 128, 129], 14, 2, 128, 24),
    ([5, -1, 300, 0, 77], 16, 2, 68, 64), ([1000, 3, -7, 250], 30, 2, 128, 128),
    ([700, 1], 16, 1, 80, 7), ([130, 64], 33, 1, 96, 5), ([200, 90], 48, 2, 32, 16),
    ([260], 9, 1, 4, 32), ([100, 200], 12, 12, 36, 64), ([333, 20], 4, 2, 124, 16), ([4000], 1, 1, 64, 256),
    ([2500, 17, 900], 32, 4, 68, 64), ([9000], 2, 2, 128, 64),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,ps", CASES)
@pytest.mark.parametrize("pad", [0, 4])
def test_step_matches_formula(cuda_device, lens, Hq, Hkv, D, ps, pad):
    s = make(cuda_device, lens, Hq, Hkv, D, ps, pad=pad)
    kp0, xp0 = s["kp"].clone(), s["xp"].clone()
    o, xn = run_step(s)
    assert o.shape == (len(lens), 1, Hq, D) and xn.shape == (len(lens), Hkv, 1, D)
    # the new row is in its page, every other element is as it was
    for b, n in enumerate(lens):
        if n >= 0:
            p = int(s["table"][b, n // ps])
            assert torch.equal(s["kp"][p, :, n % ps], s["k"][b, :, 0]) and torch.equal(s["xp"][p, :, n % ps], xn[b, :, 0])
            kp0[p, :, n % ps], xp0[p, :, n % ps] = s["k"][b, :, 0], xn[b, :, 0]
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert same(s["kp"], kp0) and same(s["xp"], xp0)
    check_step(s, o, xn)
    _lib.check_status()


@pytest.mark.parametrize("lens,Hq,Hkv,D,ps", CASES)
@pytest.mark.parametrize("pad", [0, 4])
def test_attention_matches_formula(cuda_device, lens, Hq, Hkv, D, ps, pad):
    s = make(cuda_device, lens, Hq, Hkv, D, ps, seed=1, pad=pad)
    check_attention(s, run_attention(s))
    _lib.check_status()


def test_many_sequences(cuda_device):
    """More sequences than a warp scans at once, most of them short, some unused."""
    g = np.random.default_rng(3)
    lens = [int(n) for n in g.integers(-1, 90, 150)]
    lens[70] = 4000
    s = make(cuda_device, lens, 4, 2, 64, 16, seed=2)
    check_step(s, *run_step(s))
    s = make(cuda_device, lens, 16, 1, 64, 16, seed=3)
    check_attention(s, run_attention(s))


def test_append_flag_and_two_calls(cuda_device):
    """append=False leaves the pools alone; two calls give the same bits, as do the
    appending call and the next one over the same lengths."""
    s = make(cuda_device, [500, 0, 64], 8, 2, 68, 16)
    kp0 = s["kp"].clone()
    a = run_step(s, append=False)
    assert torch.equal(s["kp"].view(torch.int16), kp0.view(torch.int16))
    b, c = run_step(s), run_step(s)
    assert all(torch.equal(x, y) for t in (b, c) for x, y in zip(a, t))


def test_step_then_attention_sees_the_new_token(cuda_device):
    """The attention over lengths + 1 after an appending step gives the step's own output
    to within the roundings of both."""
    s = make(cuda_device, [300, 1, 63], 8, 2, 128, 16)
    o, xn = run_step(s)
    s["lens"] += 1
    o2 = run_attention(s)
    check_attention(s, o)
    check_attention(s, o2)


def test_strides_and_layouts(cuda_device):
    """Operands as the projections give them, pools [P, ps, Hkv, D] seen as [P, Hkv, ps, D],
    tables that are slices of wider ones, odd starts that need a copy of the operand."""
    s = make(cuda_device, [200, 33], 8, 2, 64, 16)
    want = run_step(s, append=False)
    t = dict(s)
    t["q"] = s["q"].transpose(1, 2).contiguous().transpose(1, 2)
    t["kp"], t["xp"] = (p.transpose(1, 2).contiguous().transpose(1, 2) for p in (s["kp"], s["xp"]))
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=cuda_device)
    wide[:, 3:3 + s["table"].shape[1]] = s["table"]
    t["table"] = wide[:, 3:3 + s["table"].shape[1]]
    odd = torch.empty(2 * 8 * 64 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(2, 8, 1, 64)
    odd.copy_(s["q"])
    for other in (t, dict(s, q=odd), dict(s, v=s["v"].expand(2, 2, 1, 64))):
        got = run_step(other, append=False)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    # one row for all heads, by stride 0
    e = dict(s, q=s["q"][:, :1].expand(2, 8, 1, 64))
    check_step(e, *run_step(e, append=False))


def test_a_key_of_any_size(cuda_device):
    """Large and tiny keys: the update normalises them, the attention does not.  With
    |s q.k| up to 3e4 the softmax picks single tokens; a zero key's norm is sqrt(eps)."""
    s = make(cuda_device, [130], 4, 2, 64, 16)
    for p in s["table"][0, :9].tolist():
        s["kp"][p, 0] *= 1000
        s["kp"][p, 1] *= 1e-4
    s["k"][:, 0] *= 1000
    s["k"][:, 1] = 0
    o, xn = run_step(s, append=False)
    ref, mag = ref_update(s, 0)
    check(xn[0], ref, (2.0 ** -14 + 9 * 2.0 ** -23 * 16) * mag)
    # head 1's scores are tiny: the general bound holds there
    ref, mag, A = ref_attention(s, 0, (s["k"][0], xn[0]))
    check(o[0, 0, 2:], ref[2:], ((2.0 ** -15 + 18 * 2.0 ** -23 * A) * mag)[2:])
    assert torch.isfinite(o).all()


def test_infinite_and_nan_rows_stay_in_their_sequence(cuda_device):
    """A NaN in one sequence's cached row spoils that sequence and head only."""
    s = make(cuda_device, [100, 100], 4, 2, 64, 16)
    want, wx = run_step(s, append=False)
    s["xp"][int(s["table"][0, 2]), 1, 3, 5] = float("nan")
    s["kp"][int(s["table"][0, 3]), 1, 3, 5] = float("inf")
    o, xn = run_step(s, append=False)
    assert torch.isnan(o[0, 0, 2:]).any() and torch.equal(o[0, 0, :2], want[0, 0, :2])
    assert torch.equal(o[1], want[1]) and torch.equal(xn[1], wx[1]) and torch.equal(xn[0, 0], wx[0, 0])


def test_bad_tables_are_reported_not_followed(cuda_device):
    s = make(cuda_device, [100, 40], 4, 2, 64, 16)
    good = s["table"].clone()
    want = run_step(s, append=False)
    P = s["kp"].shape[0]
    for bad in (P, -3, 2 ** 31 - 1):
        s["table"] = good.clone()
        s["table"][0, 2] = bad
        o, _ = run_step(s, append=False)
        with pytest.raises(_lib.LucidError, match="paged decoding: a page of the block table"):
            _lib.check_status()
        assert torch.equal(o[1], want[0][1])
    # the page of the new row is missing
    s["table"] = good.clone()
    s["table"][1, 2] = -1
    before = s["kp"].clone()
    run_step(s)
    with pytest.raises(_lib.LucidError, match="a page of the block table"):
        _lib.check_status()
    n = int(s["lens"][0])
    p = int(good[0, n // 16])
    before[p, :, n % 16] = s["k"][0, :, 0]
    assert torch.equal(s["kp"].view(torch.int16), before.view(torch.int16))
    # longer than the table, and a new row just past it
    s["table"] = good
    for lens in ([good.shape[1] * 16 + 1, 40], [2 ** 31 - 1, 40]):
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
        o, xn = run_step(s, append=False)
        assert torch.equal(o[1], want[0][1]) and not o[0].any()
        with pytest.raises(_lib.LucidError, match="past the block table"):
            run_attention(s)                      # the next call says what the last one met
        run_attention(s)
        with pytest.raises(_lib.LucidError, match="past the block table"):
            _lib.check_status()
    s = make(cuda_device, [32], 4, 2, 64, 16, room=0)
    s["table"] = s["table"][:, :2].contiguous()
    run_step(s, append=False)
    _lib.check_status()
    run_step(s)
    with pytest.raises(_lib.LucidError, match="past the block table"):
        lb.copy_pages(s["kp"], s["xp"], [], []) or _lib.check_status()
    _lib.check_status()


def test_refusals(cuda_device):
    s = make(cuda_device, [20, 20], 4, 2, 64, 16)
    two = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=cuda_device)
    for kw, err in ((dict(q=two), ValueError), (dict(q=s["q"].float()), TypeError), (dict(k=s["k"][:1]), ValueError),
                    (dict(v=s["v"].half()), TypeError), (dict(table=s["table"].long()), TypeError),
                    (dict(table=s["table"][:1]), ValueError), (dict(lens=s["lens"].cpu()), ValueError),
                    (dict(lens=s["lens"][:1]), ValueError), (dict(xp=s["xp"][:, :1]), ValueError),
                    (dict(kp=s["kp"].transpose(2, 3)), ValueError), (dict(kp=s["kp"].float()), TypeError),
                    (dict(table=s["table"].t().contiguous().t()), ValueError),
                    (dict(kp=s["kp"][0].expand_as(s["kp"])), ValueError), (dict(q=s["q"][:, :3]), _lib.LucidError)):
        with pytest.raises(err):
            run_step(dict(s, **kw))
    odd = torch.zeros(5, 2, 16, 66, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="multiples of 4"):
        lb.paged_decode_attention(two[:, :, :1], odd[..., :64], odd[..., :64], s["table"], s["lens"], 0.1)
    empty = lb.paged_decode_attention(s["q"][:0], s["kp"], s["xp"], s["table"][:0], s["lens"][:0], 0.1)
    assert empty.shape == (0, 1, 4, 64)


def test_graph_replays_follow_the_lengths(cuda_device):
    """A captured step reads tables and lengths at replay, two captured graphs keep their
    own workspaces, and both replay at once on two streams."""
    a, b = make(cuda_device, [100, 3], 8, 2, 68, 16, seed=4, room=40), make(cuda_device, [70, 900], 8, 2, 68, 16, seed=5, room=40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for s in (a, b):
            run_step(s, append=False)
    torch.cuda.current_stream().wait_stream(side)
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run_step(s)
            s["lens"] += 1
        graphs.append((g, out))
    for _ in range(30):
        wants = []
        for s in (a, b):
            wants.append([t.clone() for t in run_step(s, append=False)])
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, wants):
            assert all(torch.equal(x, y) for x, y in zip(out, want))
    assert a["lens"].tolist() == [130, 33] and b["lens"].tolist() == [100, 930]
    check_step(a, *run_step(a, append=False))
    _lib.check_status()


def test_a_capture_may_be_the_first_call(cuda_device):
    """In a fresh process, with nothing called before the capture."""
    code = """
import sys; sys.path.insert(0, 'tests')
import torch, lucid_b200 as lb, test_paged_gpu as T
s = T.make('cuda', [100, 3], 8, 2, 68, 16)
x = torch.randn(4, 500, device='cuda'); t = torch.zeros(4, dtype=torch.int64, device='cuda')
k = torch.ones(2, 2, 1, 68, dtype=torch.bfloat16, device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    o, xn = T.run_step(s, append=False)
    lb.paged_append(k, k, s['kp'], s['xp'], s['table'], s['lens'])
    said = lb.token_logprobs(x, t, top=3)
g.replay(); torch.cuda.synchronize()
T.check_step(s, o, xn)
assert torch.equal(said.top_tokens, x.topk(3).indices)
assert all((s['kp'][int(s['table'][b, n // 16]), :, n % 16] == 1).all() for b, n in enumerate((100, 3)))
lb.check_status()
print('fine')
"""
    import subprocess
    import sys

    from conftest import ROOT
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip().endswith("fine"), got.stderr[-2000:]


def test_two_streams_at_once(cuda_device):
    s = [make(cuda_device, [4000, 100], 8, 2, 128, 64, seed=i) for i in range(2)]
    want = [run_step(x, append=False) for x in s]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in s], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run_step(s[i], append=False))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for out in got[i] for x, y in zip(out, want[i]))


def test_offsets_past_32_bits(cuda_device):
    """A pool of more than 2^31 elements, the sequences' pages at its end."""
    ps, D, H = 64, 128, 1
    P = 2 ** 31 // (ps * D * H) + 40
    kp = torch.empty(P, H, ps, D, dtype=torch.bfloat16, device=cuda_device)
    xp = torch.empty_like(kp)
    small = make(cuda_device, [400, 9], 4, H, D, ps)
    n = small["kp"].shape[0]
    kp[-n:], xp[-n:] = small["kp"], small["xp"]
    big = dict(small, kp=kp, xp=xp, table=torch.where(small["table"] < 0, -1, small["table"] + (P - n)).int())
    want, got = run_step(small), run_step(big)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(kp[-n:].view(torch.int16), small["kp"].view(torch.int16))
    lb.copy_pages(kp, xp, [P - 1, P - 2], [0, 1])
    assert torch.equal(kp[0].view(torch.int16), kp[-1].view(torch.int16))
    new = torch.randn(2, H, 3, D, device=cuda_device).bfloat16()
    lens = small["lens"] + 1
    lb.paged_append(new, new, kp, xp, big["table"], lens)
    lb.paged_append(new, new, small["kp"], small["xp"], small["table"], lens)
    assert torch.equal(xp[-n:].view(torch.int16), small["xp"].view(torch.int16))
    _lib.check_status()


# ---------------------------------------------------------------------------
# append and copies: exact
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("D,ps,pad", [(64, 16, 0), (68, 1, 0), (128, 24, 0), (64, 16, 4), (4, 64, 0)])
def test_append_is_exact(cuda_device, D, ps, pad):
    lens, counts, N, H = [0, 5, 33, -1, 16, 7], [9, 0, 40, 9, 1, 55], 50, 3
    s = make(cuda_device, lens, H, H, D, ps, pad=pad, room=N)
    for view in (False, True):
        g = torch.Generator(device=cuda_device).manual_seed(8 + view)
        k, x = (torch.randn(len(lens), N, H, D, generator=g, device=cuda_device).bfloat16().transpose(1, 2) for _ in range(2))
        if not view:
            k, x = k.contiguous(), torch.cat([x, x], -1)[..., :D]
        want = [p.clone() for p in (s["kp"], s["xp"])]
        for b, (n, c) in enumerate(zip(lens, counts)):
            for i in range(min(c, N) if n >= 0 else 0):
                p = int(s["table"][b, (n + i) // ps])
                want[0][p, :, (n + i) % ps], want[1][p, :, (n + i) % ps] = k[b, :, i], x[b, :, i]
        lb.paged_append(k, x, s["kp"], s["xp"], s["table"], s["lens"], torch.tensor(counts, dtype=torch.int32, device=cuda_device))
        for got, w in zip((s["kp"], s["xp"]), want):
            assert torch.equal(got.contiguous().view(torch.int16), w.contiguous().view(torch.int16))
    _lib.check_status()
    # without counts: every row of every sequence in use
    lb.paged_append(k[:, :, :2], x[:, :, :2], s["kp"], s["xp"], s["table"], s["lens"])
    assert torch.equal(s["kp"][int(s["table"][1, 5 // ps]), :, 5 % ps], k[1, :, 0])
    _lib.check_status()


def test_append_reports_and_refuses(cuda_device):
    s = make(cuda_device, [30, 2], 2, 2, 64, 16)
    k = torch.ones(2, 2, 60, 64, dtype=torch.bfloat16, device=cuda_device)
    before = s["kp"].clone()
    for counts, match in (([0, 50], "page of the block table"), ([60, 0], "past the block table")):
        lb.paged_append(k, k, s["kp"], s["xp"], s["table"], s["lens"], torch.tensor(counts, dtype=torch.int32, device=cuda_device))
        with pytest.raises(_lib.LucidError, match="a page of the block table|past the block table"):
            _lib.check_status()
    p = int(s["table"][1, 0])
    assert (s["kp"][p, :, 2:] == 1).all()          # what has a page is written
    others = [i for i in range(before.shape[0]) if i not in s["table"].unique().tolist()]
    assert torch.equal(s["kp"][others].view(torch.int16), before[others].view(torch.int16))
    for bad in (k[:1], k[:, :1], k[..., :32]):
        with pytest.raises(ValueError):
            lb.paged_append(k, bad, s["kp"], s["xp"], s["table"], s["lens"])
    with pytest.raises(TypeError):
        lb.paged_append(k, k.half(), s["kp"], s["xp"], s["table"], s["lens"])
    with pytest.raises(TypeError):
        lb.paged_append(k, k, s["kp"], s["xp"], s["table"], s["lens"], torch.ones(2, device=cuda_device))
    lb.paged_append(k[:, :, :0], k[:, :, :0], s["kp"], s["xp"], s["table"], s["lens"])
    grad = torch.ones(2, 2, 1, 64, dtype=torch.bfloat16, device=cuda_device, requires_grad=True)
    lb.paged_append(grad, grad, s["kp"], s["xp"], s["table"], s["lens"])
    assert not s["kp"].requires_grad
    _lib.check_status()


@pytest.mark.parametrize("shape", [(40, 2, 16, 64), (3, 1000, 1, 1, 4), (2, 40, 3, 24, 68), (5, 12, 1, 5, 12)])
def test_copy_pages_is_exact(cuda_device, shape):
    g = torch.Generator(device=cuda_device).manual_seed(1)
    k, x = (torch.randn(*shape, generator=g, device=cuda_device).bfloat16() for _ in range(2))
    P = shape[-4]
    order = torch.randperm(P, generator=torch.Generator().manual_seed(2))
    half = P // 2
    src, dst = order[:half], order[half:2 * half]
    src[0] = src[-1]                                   # one page copied to two places
    want = []
    for t in (k, x):
        w = t.clone()
        (w if len(shape) == 4 else w.transpose(0, 1))[dst.to(cuda_device)] = (t if len(shape) == 4 else t.transpose(0, 1))[src.to(cuda_device)]
        want.append(w)
    # the values' pool in another order of its inner dimensions: still dense pages
    x2 = x.transpose(-3, -2).contiguous().transpose(-3, -2)
    lb.copy_pages(k, x2, src, dst.tolist())
    assert torch.equal(k, want[0]) and torch.equal(x2, want[1])


def test_copy_pages_refusals(cuda_device):
    k = torch.zeros(6, 2, 4, 8, dtype=torch.bfloat16, device=cuda_device)
    for src, dst in (([0], [6]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            lb.copy_pages(k, k.clone(), src, dst)
    with pytest.raises(TypeError):
        lb.copy_pages(k, k.clone(), torch.tensor([0], device=cuda_device), [1])
    with pytest.raises(ValueError, match="dense"):
        wide = torch.zeros(6, 2, 4, 16, dtype=torch.bfloat16, device=cuda_device)[..., :8]
        lb.copy_pages(wide, k, [0], [1])
    lb.copy_pages(k, k.clone(), [], [])
    _lib.check_status()


def test_copy_pages_in_a_graph(cuda_device):
    k = torch.randn(8, 2, 4, 8, device=cuda_device).bfloat16()
    x = k.clone()
    g = torch.cuda.CUDAGraph()
    lb.copy_pages(k, x, [7], [6])
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        lb.copy_pages(k, x, [0, 1], [2, 3])            # the pairs are the launch's own
    k[0] = 5
    g.replay()
    assert (k[2] == 5).all() and torch.equal(k[3], k[1])


# ---------------------------------------------------------------------------
# together, as a server uses them
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def model():
    from lucid_b200.decoder import LucidForCausalLM, lucid_config
    cfg = lucid_config(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=8,
                       num_key_value_heads=1, head_dim=68, vocab_size=1000)
    return LucidForCausalLM(cfg).to("cuda", torch.bfloat16).init_weights(seed=3, std=0.05).eval()


def _dense_logits(model, prompt, tokens):
    """Logits of every new token through the dense transformers cache, token by token."""
    from transformers import DynamicCache
    with torch.no_grad():
        cache, out = DynamicCache(), []
        logits = model(prompt[None], past_key_values=cache, logits_to_keep=1)
        for t in tokens:
            out.append(logits[0, -1].float())
            logits = model(t.view(1, 1), past_key_values=cache)
    return torch.stack(out)


def test_generation_over_pages_matches_the_dense_cache(cuda_device, model):
    """Ragged prompts, right-padded: the paged run's tokens are scored again one prompt at a
    time over the dense cache.  Bound as for the dense cache against the fused prefill
    (two bf16 paths through the same model)."""
    g = torch.Generator().manual_seed(4)
    lens, new = [130, 1, 57], 12
    ids = torch.randint(0, 1000, (3, max(lens)), generator=g).to(cuda_device)
    cache = lb.PagedCache.for_config(model.config, num_pages=40, page_size=16)
    batch = cache.batch(cache.new(3))
    tokens, said = model.generate(ids, batch, new, prompt_lengths=lens, top=3)
    assert tokens.shape == (3, new) and said.logprobs.shape == (3, new) and said.top_tokens.shape == (3, new, 3)
    assert batch.host_lengths == [n + new - 1 for n in lens] and batch.lengths.tolist() == batch.host_lengths
    assert torch.equal(said.top_tokens[..., 0], tokens)
    for b, n in enumerate(lens):
        logits = _dense_logits(model, ids[b, :n], tokens[b])
        lp = torch.log_softmax(logits, -1)
        scale = logits.abs().max().item()
        assert (lp.gather(1, tokens[b][:, None])[:, 0] - said.logprobs[b]).abs().max().item() <= 3e-2 * scale
        assert (-(lp.exp() * lp).sum(-1) - said.entropy[b]).abs().max().item() <= 3e-2 * scale
    _lib.check_status()


def test_forking_freeing_and_compacting_keep_the_tokens(cuda_device, model):
    """Logits do not change when pages move, and a fork goes on like its parent."""
    cache = lb.PagedCache.for_config(model.config, num_pages=60, page_size=16)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 1000, (4, 37), generator=g).to(cuda_device)
    seqs = cache.new(4)
    with torch.no_grad():
        model(ids, cache.batch(seqs))
        cache.free(seqs[0])
        cache.free(seqs[2])
        child = cache.fork(seqs[3])
        nxt = torch.randint(0, 1000, (3, 1), generator=g).to(cuda_device)
        nxt[2] = nxt[1]                                   # parent and child read the same token
        rest = cache.batch([seqs[1], seqs[3], child])
        held = {s: [[t[:, p].clone() for p in cache.pages(s)] for t in (cache.key_pages, cache.x_pages)] for s in rest.sequences}
        a = model(nxt, rest)
        # rows differ only in how the batch's tiles were dealt out: fp32 join order, then bf16
        assert (a[1] - a[2]).abs().max().item() <= 2e-2 * a.float().abs().max().item()
        assert cache.pages(seqs[3])[:2] == cache.pages(child)[:2] and cache.pages(seqs[3])[2] != cache.pages(child)[2]
        for s, pools in held.items():                     # the tokens cached before are where the list says
            for was, pool in zip(pools, (cache.key_pages, cache.x_pages)):
                for i, (old, p) in enumerate(zip(was, cache.pages(s))):
                    rows = min(16, 37 - 16 * i)
                    assert torch.equal(pool[:, p, :, :rows], old[:, :, :rows])
        nxt = torch.randint(0, 1000, (3, 1), generator=g).to(cuda_device)
        lens = [cache.length(s) for s in rest.sequences]
        b = model(nxt, rest)
        for s, n in zip(rest.sequences, lens):            # the same step again, after moving pages
            cache._sequences[s].length = n
        assert cache.compact() > 0
        used = {p for s in rest.sequences for p in cache._sequences[s].pages}
        assert used == set(range(len(used)))
        c = model(nxt, cache.batch(rest.sequences))
    assert torch.equal(b, c)
    _lib.check_status()


def test_a_captured_step_and_stale_batches(cuda_device, model):
    cache = lb.PagedCache.for_config(model.config, num_pages=20, page_size=16)
    batch = cache.batch(cache.new(2))
    ids = torch.zeros(2, 5, dtype=torch.int64, device=cuda_device)
    with torch.no_grad():
        model(ids, batch)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with pytest.raises(_lib.LucidError, match="before the capture"):
            with torch.cuda.graph(g):
                model(ids[:, :1], batch)
        torch.cuda.synchronize()
        logits = model(ids[:, :1], batch)
    assert torch.isfinite(logits).all() and batch.host_lengths == [6, 6]


def test_score_matches_log_softmax(cuda_device, model):
    ids = torch.randint(0, 1000, (2, 64), generator=torch.Generator().manual_seed(6)).to(cuda_device)
    said = model.score(ids, top=4)
    with torch.no_grad():
        lp = torch.log_softmax(model(ids)[:, :-1].double(), -1)
    assert (said.logprobs - lp.gather(2, ids[:, 1:, None])[..., 0]).abs().max().item() < 1e-5
    assert (said.top_logprobs - lp.topk(4).values).abs().max().item() < 1e-5
    assert (said.entropy + (lp.exp() * lp).sum(-1)).abs().max().item() < 1e-5
