"""The language-model operators against plain implementations in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of float32, in which the operators compute; h(type) half a step of
the result's type, relative to the value.
  embedding            one product (u), one rounding (h)
  embedding_grad       a sum of c terms (at most c + 2 roundings of the sum of absolute values: join, scale), one rounding (h)
  gated_scan           each token's gate and its complement are off by a relative e = (12 + 4 |gate|) u at most (argument of
                       the exponential, exponential, sum, reciprocal, product), each step rounds twice more; the error then
                       obeys the recurrence E[t] = f E[t-1] + (e + 4 u) H[t] with H the recurrence of absolute values;
                       joining runs, warps and blocks adds at most 40 roundings of H per token; one rounding (h).  A product
                       below the normal range is off by half a denormal step, 2^-150, whatever its size: 4 + 40 of them per
                       token, so E[t] gains 44 * 2^-150 beside the relative terms (a state that has decayed that far)
  token_logprobs       exponents of up to 30 (smaller weights do not count) times 2 u and two units for the exponential,
                       sums of `adds` terms per thread and 40 joins: (80 + adds) u absolute in log2, a few u relative
"""
import math

import numpy as np
import pytest

import appy_b200 as appy

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOST = 44 * 2.0 ** -150
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):                                   # below the normal range a result is off by half a denormal step
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(*shape, dtype=torch.float32, seed=0, std=1.0, mean=0.0):
    return torch.empty(*shape, device="cuda").normal_(mean, std, generator=gen(seed)).to(dtype)


def within(got, ref, tol):
    got = got.double()
    assert got.shape == ref.shape
    same = (got == ref) | (got.isnan() & ref.isnan())
    off = torch.where(same, 0.0, (got - ref).abs())
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off - tol).nan_to_num(math.inf).max())}"


# ------------------------------------------------------------------------------------------------ embedding

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 7, 8, 64, 100, 769, 1024, 2056])
@pytest.mark.parametrize("n", [0, 1, 33, 1000])
def test_embedding(rt, dtype, width, n):
    rows = 517
    w = randn(rows, width, dtype=dtype, seed=width)
    tokens = torch.randint(-3, rows + 3, (n,), generator=gen(n), device="cuda", dtype=torch.int32 if width % 2 else torch.int64)
    known = (tokens >= 0) & (tokens < rows)
    exact = torch.where(known[:, None], w.double()[torch.where(known, tokens, 0).long()], 0.0)
    got = appy.embedding(w, tokens)
    assert got.dtype == dtype and torch.equal(got.double(), exact)
    ref = exact * float(np.float32(0.7))
    within(appy.embedding(w, tokens, scale=0.7), ref, (U + half(dtype)) * ref.abs() * 1.01 + tiny(dtype))


def test_embedding_strides_shapes_and_out(rt):
    w = randn(100, 96, dtype=torch.bfloat16, seed=1)
    tokens = torch.randint(0, 100, (3, 5), generator=gen(2), device="cuda")
    ref = w[tokens]
    assert torch.equal(appy.embedding(w, tokens), ref)
    assert torch.equal(appy.embedding(w[:, 8:72], tokens), ref[..., 8:72])          # rows of a wider table
    assert torch.equal(appy.embedding(w[:, 3:70], tokens), ref[..., 3:70])          # rows that start off 16 bytes
    assert torch.equal(appy.embedding(w[::2], tokens // 2), w[::2][tokens // 2])
    assert torch.equal(appy.embedding(w.t().contiguous().t(), tokens), ref)          # columns apart: copied first
    assert torch.equal(appy.embedding(w, tokens.t()), w[tokens.t()])
    buffer = torch.full((3, 5, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    out = appy.embedding(w, tokens, out=buffer[..., 16:112])
    assert out.data_ptr() == buffer[..., 16:112].data_ptr() and torch.equal(buffer[..., 16:112], ref)
    assert (buffer[..., :16] == 9).all() and (buffer[..., 112:] == 9).all()
    one = torch.tensor(7, device="cuda")
    assert torch.equal(appy.embedding(w, one), w[7])
    assert appy.embedding(w[:0], tokens).abs().max() == 0


# ------------------------------------------------------------------------------------------------ embedding gradient

def grad_reference(grad, tokens, rows, scale=1.0):
    known = (tokens >= 0) & (tokens < rows)
    t, g = tokens[known].long(), grad.double()[known] * float(np.float32(scale))
    total = torch.zeros(rows, grad.shape[-1], dtype=torch.float64, device="cuda").index_add_(0, t, g)
    size = torch.zeros_like(total).index_add_(0, t, g.abs())
    count = torch.zeros(rows, 1, dtype=torch.float64, device="cuda").index_add_(0, t, torch.ones(len(t), 1, dtype=torch.float64, device="cuda"))
    return total, size, count


def grad_tolerance(ref, size, count, dtype):
    return (count + 3) * U * size + half(dtype) * (ref.abs() + (count + 3) * U * size) + tiny(dtype)


def draw_tokens(kind, n, rows, seed):
    if kind == "uniform":
        return torch.randint(0, rows, (n,), generator=gen(seed), device="cuda")
    if kind == "zipf":
        return (torch.exp(torch.rand(n, generator=gen(seed), device="cuda") * math.log(rows + 1)) - 1).long().clamp(0, rows - 1)
    if kind == "one":
        return torch.full((n,), rows // 2, device="cuda")
    if kind == "two":                                   # the first and the last row
        return torch.randint(0, 2, (n,), generator=gen(seed), device="cuda") * (rows - 1)
    if kind == "none":
        return torch.where(torch.rand(n, generator=gen(seed), device="cuda") < 0.5, -1, rows)
    return torch.arange(n, device="cuda").flip(0) % rows


@pytest.mark.parametrize("dtype, out_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                              (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("n, rows, width", [(1, 1, 1), (1, 1000, 64), (31, 5, 8), (33, 511, 769), (256, 90, 24), (257, 90, 24), (700, 512, 100), (4096, 513, 256), (4097, 100, 40),
                                            (9000, 70001, 72), (20011, 300, 264)])
def test_embedding_grad(rt, dtype, out_dtype, n, rows, width):
    for k, kind in enumerate(["uniform", "zipf", "one", "two", "none", "falling"]):
        tokens = draw_tokens(kind, n, rows, seed=n + k)
        if k == 1:
            tokens = torch.where(torch.rand(n, generator=gen(5), device="cuda") < 0.2, -100, tokens)
        tokens = tokens.to(torch.int32 if k % 2 else torch.int64)
        grad = randn(n, width, dtype=dtype, seed=k)
        out = torch.full((rows, width), float("nan"), dtype=out_dtype, device="cuda")
        got = appy.embedding_grad(grad, tokens, scale=0.3, out=out)
        ref, size, count = grad_reference(grad, tokens, rows, 0.3)
        assert got is out
        within(got, ref, grad_tolerance(ref, size, count, out_dtype))
        assert not got[count[:, 0] == 0].any()
        again = appy.embedding_grad(grad, tokens, scale=0.3, out=torch.empty_like(out))
        assert torch.equal(got, again)                  # the same bits whatever the schedule


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_embedding_grad_accumulates_and_leaves_other_rows(rt, dtype):
    n, rows, width = 3000, 5000, 136
    tokens = draw_tokens("zipf", n, rows, 3)
    grad = randn(n, width, dtype=torch.bfloat16 if dtype == torch.bfloat16 else dtype, seed=4)
    wide = randn(rows, 2 * width, dtype=dtype, seed=5)
    before = wide.clone()
    out = wide[:, 24:24 + width]                        # rows of a wider array
    appy.embedding_grad(grad, tokens, out=out, accumulate=True)
    ref, size, count = grad_reference(grad, tokens, rows)
    old = before[:, 24:24 + width].double()
    ref2 = ref + old
    within(out, ref2, grad_tolerance(ref2, size + old.abs(), count + 1, dtype))
    assert torch.equal(wide[:, :24], before[:, :24]) and torch.equal(wide[:, 24 + width:], before[:, 24 + width:])
    assert torch.equal(out[count[:, 0] == 0], before[:, 24:24 + width][count[:, 0] == 0])


def test_embedding_grad_of_broadcast_and_strided_gradients(rt):
    tokens = torch.randint(0, 50, (4, 9), generator=gen(1), device="cuda")
    ones = torch.ones((), device="cuda").expand(4, 9, 24)               # what a sum hands back
    ref, size, count = grad_reference(torch.ones(36, 24, device="cuda"), tokens.reshape(-1), 50)
    assert torch.equal(appy.embedding_grad(ones, tokens, 50).double(), ref)
    g = randn(4, 9, 48, seed=2)
    ref, size, count = grad_reference(g[..., 8:32].reshape(36, 24), tokens.reshape(-1), 50)
    within(appy.embedding_grad(g[..., 8:32], tokens, 50), ref, grad_tolerance(ref, size, count, torch.float32))
    t = randn(24, 36, seed=3).t().reshape(4, 9, 24)
    ref, size, count = grad_reference(t.reshape(36, 24), tokens.reshape(-1), 50)
    within(appy.embedding_grad(t, tokens, 50), ref, grad_tolerance(ref, size, count, torch.float32))
    assert appy.embedding_grad(randn(0, 24), tokens[:0, 0], 7).abs().max() == 0          # no tokens: zeros
    assert appy.embedding_grad(randn(4, 9, 24), tokens, 0).shape == (0, 24)


def test_embedding_grad_of_many_positions(rt):
    n, rows, width = (1 << 20) + 77, 3001, 16           # several tiles per block of the sort, long shares
    tokens = draw_tokens("zipf", n, rows, 9).int()
    grad = randn(n, width, dtype=torch.bfloat16, seed=10)
    ref, size, count = grad_reference(grad, tokens, rows)
    within(appy.embedding_grad(grad, tokens, rows, out=torch.empty(rows, width, device="cuda")), ref, grad_tolerance(ref, size, count, torch.float32))


# ------------------------------------------------------------------------------------------------ gated recurrence

def scan_reference(x, gate, initial, lengths, firsts, grad=None, grad_last=None):
    """Sequences of x, gate [rows, width] one token after another in float64, with the error bounds of the module's docstring."""
    rows, width = x.shape
    b = len(lengths)
    n, lo = torch.tensor(lengths, device="cuda"), torch.tensor(firsts, device="cuda")
    z = lambda: torch.zeros(rows, width, dtype=torch.float64, device="cuda")  # noqa: E731
    f, i = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    e = (16 + 4 * gate.double().abs().clamp_max(200)) * U
    h0 = initial.double() if initial is not None else torch.zeros(b, width, dtype=torch.float64, device="cuda")
    h, H, E = z(), z(), z()
    s, S, Es = h0.clone(), h0.abs(), torch.zeros_like(h0)
    longest = max(lengths, default=0)
    for t in range(longest):
        on = (n > t).nonzero()[:, 0]
        at = lo[on] + t
        s[on] = f[at] * s[on] + i[at] * x[at].double()
        S[on] = f[at] * S[on] + i[at] * x[at].double().abs()
        Es[on] = f[at] * Es[on] + e[at] * S[on] + LOST
        h[at], H[at], E[at] = s[on], S[on], Es[on]
    out = {"h": h, "h_tol": E + 40 * U * H, "last": s, "last_tol": Es + 40 * U * S, "H": H}
    if grad_last is None:
        return out
    lam, L, El = grad_last.double(), grad_last.double().abs(), torch.zeros_like(h0)
    dx, dg, dx_tol, dg_tol = z(), z(), z(), z()
    type_half = half(x.dtype)
    for t in reversed(range(longest)):
        on = (n > t).nonzero()[:, 0]
        at = lo[on] + t
        before = h0[on] if t == 0 else h[at - 1]
        before_tol = torch.zeros_like(before) if t == 0 else out["h_tol"][at - 1] + type_half * (h[at - 1].abs() + out["h_tol"][at - 1]) + tiny(x.dtype)
        g = grad[at].double() if grad is not None else torch.zeros_like(before)
        lam[on], L[on] = lam[on] + g, L[on] + g.abs()
        err = El[on] + 40 * U * L[on] + LOST
        dx[at] = lam[on] * i[at]
        dx_tol[at] = (err + e[at] * L[on]) * i[at]
        fi, diff, wide = f[at] * i[at], before - x[at].double(), before.abs() + x[at].double().abs()
        dg[at] = lam[on] * diff * fi
        dg_tol[at] = err * wide * fi + L[on] * (before_tol + (2 * e[at] + 4 * U) * wide) * fi
        lam[on], L[on] = lam[on] * f[at], L[on] * f[at]
        El[on] = f[at] * El[on] + e[at] * L[on] + LOST
    out.update(dx=dx, dx_tol=dx_tol, dg=dg, dg_tol=dg_tol, d0=lam, d0_tol=El + 40 * U * L)
    return out


def rounded(ref, tol, dtype):
    return tol + half(dtype) * (ref.abs() + tol) + tiny(dtype)


def check_scan(x, gate, initial, offsets, lengths, firsts, with_grad=True, seed=0, with_dh=True):
    rows, width = x.numel() // x.shape[-1], x.shape[-1]
    flat = lambda t: t.reshape(rows, width)  # noqa: E731
    covered = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, n in zip(firsts, lengths):
        covered[a:a + n] = True
    dh = randn(*x.shape, dtype=x.dtype, seed=seed + 1) if with_dh else None
    dl = randn(len(lengths), width, seed=seed + 2)
    ref = scan_reference(flat(x), flat(gate), initial, lengths, firsts, flat(dh) if with_dh else None, dl)
    h, last = appy.gated_scan(x, gate, initial, offsets)
    assert h.dtype == x.dtype and last.dtype == torch.float32 and h.shape == x.shape
    within(flat(h), ref["h"], rounded(ref["h"], ref["h_tol"], x.dtype))
    within(last, ref["last"], ref["last_tol"] + U * ref["last"].abs())
    assert not flat(h)[~covered].any()
    if not with_grad:
        return
    dx, dg, d0 = appy.gated_scan_grad(dh, x, gate, h, initial, offsets, dl)
    within(flat(dx), ref["dx"], rounded(ref["dx"], ref["dx_tol"], x.dtype))
    within(flat(dg), ref["dg"], rounded(ref["dg"], ref["dg_tol"], x.dtype))
    within(d0, ref["d0"], ref["d0_tol"] + U * ref["d0"].abs())
    assert not flat(dx)[~covered].any() and not flat(dg)[~covered].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch, tokens, width", [(1, 1, 1), (3, 1, 64), (2, 2, 4), (5, 7, 33), (1, 127, 64), (2, 128, 68), (1, 129, 100), (3, 300, 130),
                                                  (1, 1025, 64), (2, 1500, 12), (1, 3000, 3)])
def test_gated_scan_dense(rt, dtype, batch, tokens, width):
    x, gate = randn(batch, tokens, width, dtype=dtype, seed=1), randn(batch, tokens, width, dtype=dtype, seed=2, mean=2.0, std=2.0)
    firsts, lengths = [b * tokens for b in range(batch)], [tokens] * batch
    check_scan(x, gate, randn(batch, width, seed=3), None, lengths, firsts)
    check_scan(x, gate, None, None, lengths, firsts, with_dh=tokens % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [64, 7, 260])
@pytest.mark.parametrize("lengths, before, after", [([5], 0, 0), ([0], 0, 3), ([0, 0, 4, 0], 2, 0), ([1, 130, 0, 257, 2], 0, 5), ([1100, 1, 40], 7, 9),
                                                    ([3] * 40, 1, 1)])
def test_gated_scan_packed(rt, dtype, width, lengths, before, after):
    total = before + sum(lengths) + after
    firsts = [before + sum(lengths[:k]) for k in range(len(lengths))]
    x, gate = randn(total, width, dtype=dtype, seed=1), randn(total, width, dtype=dtype, seed=2, mean=1.0, std=2.0)
    offsets = torch.tensor(firsts + [before + sum(lengths)], dtype=torch.int32 if width % 2 else torch.int64, device="cuda")
    check_scan(x, gate, randn(len(lengths), width, seed=3), offsets, lengths, firsts)


def test_gated_scan_many_sequences_and_many_channels(rt):
    x, gate = randn(700, 9, 20, seed=1), randn(700, 9, 20, seed=2)
    check_scan(x, gate, randn(700, 20, seed=3), None, [9] * 700, [9 * b for b in range(700)])
    x, gate = randn(2, 40, 20000, dtype=torch.bfloat16, seed=1), randn(2, 40, 20000, dtype=torch.bfloat16, seed=2)
    check_scan(x, gate, randn(2, 20000, seed=3), None, [40] * 2, [0, 40])


def test_gated_scan_strides(rt):
    b, t, d = 3, 150, 72
    p = randn(b, t, 2 * d, dtype=torch.bfloat16, seed=1)                # x and gate are the halves of one projection
    x, gate = p[..., :d], p[..., d:]
    h, last = appy.gated_scan(x, gate)
    h2, last2 = appy.gated_scan(x.contiguous(), gate.contiguous())
    assert torch.equal(h, h2) and torch.equal(last, last2)
    tb = p.transpose(0, 1).contiguous().transpose(0, 1)                 # tokens first in memory
    h3, last3 = appy.gated_scan(tb[..., :d], tb[..., d:])
    assert torch.equal(h, h3) and torch.equal(last, last3)
    odd = torch.empty(b, t, 2 * d + 3, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:2 * d + 1] = p                                           # rows off every boundary
    h4, last4 = appy.gated_scan(odd[..., 1:d + 1], odd[..., d + 1:2 * d + 1])
    within(h4, h.double(), 2 * half(torch.bfloat16) * h.double().abs() + 1e-5)
    within(last4, last.double(), 1e-5 + 1e-5 * last.double().abs())
    apart = x.transpose(1, 2).contiguous().transpose(1, 2)              # channels apart: copied first
    assert torch.equal(appy.gated_scan(apart, gate)[0], h)
    dh = randn(b, t, d, dtype=torch.bfloat16, seed=5)
    dp = torch.full_like(p, 7.0)
    dx, dg, d0 = appy.gated_scan_grad(dh, x, gate, h, out=(dp[..., :d], dp[..., d:]))
    ex, eg, e0 = appy.gated_scan_grad(dh, x.contiguous(), gate.contiguous(), h)
    assert torch.equal(dp[..., :d], ex) and torch.equal(dp[..., d:], eg) and torch.equal(d0, e0)
    ones = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(b, t, d)
    for got, ref in zip(appy.gated_scan_grad(ones, x, gate, h), appy.gated_scan_grad(ones.contiguous(), x, gate, h)):
        assert torch.equal(got, ref)
    shared = x[:1].expand(b, t, d)                                      # one input for all sequences
    assert torch.equal(appy.gated_scan(shared, gate)[0], appy.gated_scan(shared.contiguous(), gate)[0])


def test_gated_scan_leaves_rows_behind_the_last_sequence(rt):
    x, gate = randn(50, 64, seed=1), randn(50, 64, seed=2)
    offsets = torch.tensor([3, 10, 41], device="cuda")
    out = torch.full((50, 64), 7.0, device="cuda")
    h, _ = appy.gated_scan(x, gate, offsets=offsets, out=out)
    assert h is out and (out[:3] == 7).all() and (out[41:] == 7).all()
    assert torch.equal(out[3:41], appy.gated_scan(x, gate, offsets=offsets)[0][3:41])
    dx, dg = torch.full_like(out, 7.0), torch.full_like(out, 7.0)
    appy.gated_scan_grad(x, x, gate, h, offsets=offsets, out=(dx, dg))
    for d in (dx, dg):
        assert (d[:3] == 7).all() and (d[41:] == 7).all() and not (d[3:41] == 7).any()
    h, last = appy.gated_scan(x, gate, offsets=torch.tensor([-5, 60], device="cuda"))      # positions outside count as the ends
    assert torch.equal(h, appy.gated_scan(x[None], gate[None])[0][0])
    h, last = appy.gated_scan(x, gate, offsets=torch.tensor([20, 10], device="cuda"), initial=x[:1])
    assert torch.equal(last, x[:1]) and not h[20:].any()


def test_gated_scan_steps_a_state_in_place(rt):
    b, t, d = 5, 6, 200
    x, gate = randn(b, t, d, dtype=torch.float16, seed=1), randn(b, t, d, dtype=torch.float16, seed=2)
    start = randn(b, d, seed=3)
    whole, last = appy.gated_scan(x, gate, start)
    state = start.clone()
    for k in range(t):
        step, out = appy.gated_scan(x[:, k:k + 1], gate[:, k:k + 1], state, last=state)
        assert out is state
        within(step, whole[:, k:k + 1].double(), 2 * half(torch.float16) * whole[:, k:k + 1].double().abs() + 1e-5)
    within(state, last.double(), 1e-5 * (1 + last.double().abs()))
    long_x, long_g = randn(2, 5000, 64, seed=4), randn(2, 5000, 64, seed=5)             # a cluster per sequence, in place
    start = randn(2, 64, seed=6)
    state = start.clone()
    _, last = appy.gated_scan(long_x, long_g, start)
    appy.gated_scan(long_x, long_g, state, last=state)
    assert torch.equal(state, last)


def test_gated_scan_closed_and_open_gates(rt):
    x, gate = randn(1, 300, 64, seed=1), torch.zeros(1, 300, 64, device="cuda")
    gate[:, :, :16] = math.inf                                           # keeps the state
    gate[:, :, 16:32] = -math.inf                                        # takes the input
    gate[:, :, 32:48] = torch.finfo(torch.float32).max
    gate[:, :, 48:] = torch.finfo(torch.float32).min
    start = randn(1, 64, seed=2)
    h, last = appy.gated_scan(x, gate, start)
    for c in (0, 32):
        assert torch.equal(h[..., c:c + 16], start[:, None, c:c + 16].expand(1, 300, 16))
        assert torch.equal(h[..., c + 16:c + 32], x[..., c + 16:c + 32])
    dx, dg, d0 = appy.gated_scan_grad(x, x, gate, h, start)
    # a closed gate counts as -87, so f (1 - f) is at most 2^-125 there; |lam| and |h - x| are below 16
    assert dg.abs().max() <= 2.0 ** -125 * 16 * 16 and not dx[..., :16].any() and torch.equal(dx[..., 16:32], x[..., 16:32])
    x[0, 100, 3] = math.nan
    h, last = appy.gated_scan(x, torch.ones_like(gate), start)
    assert h[0, 100:, 3].isnan().all() and not h[0, :100].isnan().any() and not h[..., :3].isnan().any() and not h[..., 4:].isnan().any()
    assert appy.gated_scan(x[:, :0], gate[:, :0], start)[1].equal(start)


def test_gated_scan_gradient_against_differences(rt):
    b, t, d = 2, 9, 5
    x, gate, start = randn(b, t, d, seed=1), randn(b, t, d, seed=2), randn(b, d, seed=3)
    wh, wl = randn(b, t, d, seed=4).double(), randn(b, d, seed=5).double()

    def loss(x, gate, start):
        s, total = start, 0.0
        for k in range(t):
            f = torch.sigmoid(gate[:, k])
            s = f * s + (1 - f) * x[:, k]
            total = total + (wh[:, k] * s).sum()
        return total + (wl * s).sum()

    h, _ = appy.gated_scan(x, gate, start)
    got = appy.gated_scan_grad(wh.float(), x, gate, h, start, grad_last=wl.float())
    at = [v.double() for v in (x, gate, start)]
    eps = 1e-6
    for which, g in enumerate(got):
        for k in range(0, g.numel(), 7):
            up, down = [v.clone() for v in at], [v.clone() for v in at]
            up[which].view(-1)[k] += eps
            down[which].view(-1)[k] -= eps
            assert abs(float(loss(*up) - loss(*down)) / (2 * eps) - float(g.reshape(-1)[k])) < 1e-4


# ------------------------------------------------------------------------------------------------ log probabilities

def logprob_reference(logits, tokens, temperature, top):
    z = logits.double() / float(np.float32(temperature))
    m = z.amax(-1, keepdim=True)
    empty = m == -math.inf
    d = z - torch.where(empty, 0.0, m)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logp = torch.where(empty, -math.inf, d - torch.log(total))
    p = torch.where(empty, 0.0, e / total)
    plogp = torch.where(p > 0, p * logp, torch.where(p.isnan(), p, 0.0))
    entropy = -plogp.sum(-1)
    known = (tokens >= 0) & (tokens < z.shape[-1])
    lp = torch.where(known, logp.gather(-1, torch.where(known, tokens, 0).long()[..., None])[..., 0], 0.0)
    order = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[..., :top]
    return lp, entropy, logp.gather(-1, order), order, (logp, p, plogp, empty[..., 0], known)


def logprob_tolerance(cols):
    adds = math.ceil(cols / 512)
    return (80 + adds) * U


def check_logprobs(logits, tokens, temperature=1.0, top=0, seed=0, grads="both"):
    r = appy.token_logprobs(logits, tokens, top=top, temperature=temperature)
    lp, entropy, top_lp, order, (logp, p, plogp, empty, known) = logprob_reference(logits, tokens, temperature, top)
    lp, top_lp = (torch.where(v.abs() > torch.finfo(torch.float32).max, v.float().double(), v) for v in (lp, top_lp))     # beyond float32: infinite
    cols = logits.shape[-1]
    tol = logprob_tolerance(cols)
    finite = lambda v: torch.where(v.isfinite(), v.abs(), 0.0)  # noqa: E731
    within(r.logprobs, lp, tol + 8 * U * finite(lp))
    etol = tol * (2 + math.log2(cols + 1))
    within(r.entropy, entropy, torch.full_like(entropy, etol))
    if top:
        within(r.top_logprobs, top_lp, tol + 8 * U * finite(top_lp))
        assert r.top_tokens.dtype == tokens.dtype and torch.equal(r.top_tokens.long(), order)
    else:
        assert r.top_logprobs is None and r.top_tokens is None
    g, gh = randn(*tokens.shape, seed=seed + 1), randn(*tokens.shape, seed=seed + 2)
    if grads == "logprobs":
        gh = None
    if grads == "entropy":
        g = None
    got = appy.token_logprobs_grad(logits, tokens, r.stats, g, gh, temperature)
    g64 = torch.where(known, g.double(), 0.0)[..., None] if g is not None else torch.zeros_like(lp)[..., None]
    h64 = gh.double()[..., None] if gh is not None else torch.zeros_like(lp)[..., None]
    one = torch.zeros_like(p).scatter_(-1, torch.where(known, tokens, 0).long()[..., None], known.double()[..., None])
    ref = g64 * (one - p) - h64 * (plogp + p * entropy[..., None])
    t = float(np.float32(temperature))
    ref = torch.where(empty[..., None], 0.0, ref) / t
    alogp = torch.where(p > 0, logp.abs(), 0.0)
    size = p * (g64.abs() + h64.abs() * (alogp + entropy[..., None].abs()))
    bound = (size * (tol + 16 * U + 4 * U * alogp) + p * h64.abs() * (etol + tol + 8 * U * alogp) + 4 * U * one * g64.abs()) / t
    # a probability below 2^-126 counts as zero; p |log p| is at most 88 * 2^-126 there
    bound = bound + 2.0 ** -126 * (g64.abs() + h64.abs() * (88 + entropy[..., None].abs())) / t
    bound = torch.where(empty[..., None], 0.0, bound)
    within(got, ref, bound + half(logits.dtype) * (ref.abs() + bound) + tiny(logits.dtype))
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, cols, top", [(1, 1, 1), (3, 7, 7), (5, 33, 20), (2, 1000, 32), (40, 1021, 5), (1, 4099, 20), (300, 5003, 1), (1, 50257, 32),
                                          (5, 131072, 20), (700, 520, 3)])
def test_token_logprobs(rt, dtype, n, cols, top):
    logits = randn(n, cols, dtype=dtype, seed=n, std=4.0)
    tokens = torch.randint(0, cols, (n,), generator=gen(1), device="cuda", dtype=torch.int32 if cols % 2 else torch.int64)
    check_logprobs(logits, tokens, 1.0, top)
    check_logprobs(logits, tokens, 0.6, 0, grads="logprobs")
    check_logprobs(logits, tokens, 2.5, min(top, 2), grads="entropy")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 130, 3001, 20000])
@pytest.mark.parametrize("temperature", [1.0, 0.1, 30.0])
def test_token_logprobs_masked(rt, dtype, cols, temperature):
    lowest = torch.finfo(dtype).min
    logits = randn(12, cols, dtype=dtype, seed=cols, std=2.0)
    logits[0] = -math.inf                              # nothing left
    logits[1] = lowest                                 # the type's lowest value everywhere: even
    logits[2, 1:] = -math.inf                          # one left
    logits[3, : cols // 2] = lowest
    logits[4, cols // 2:] = -math.inf
    logits[5] = lowest
    logits[5, : cols // 2] = -math.inf                 # both kinds and nothing else
    logits[6] = 0.0
    logits[6, -1] = -0.0                               # all equal, zeros of both signs
    logits[7] = torch.finfo(dtype).max
    logits[8, 3] = torch.finfo(dtype).max
    logits[9, ::2] = logits[9, 1]                      # many ties
    logits[10] = lowest
    logits[10, 5] = lowest / 2
    tokens = torch.randint(0, cols, (12,), generator=gen(2), device="cuda")
    tokens[3], tokens[4], tokens[11] = 0, cols - 1, -100
    check_logprobs(logits, tokens, temperature, min(20, cols))
    tokens[11] = cols
    check_logprobs(logits, tokens.int(), temperature, 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_token_logprobs_not_finite(rt, dtype):
    logits = randn(4, 5000, dtype=dtype, seed=3)
    logits[0, 17], logits[1, 4999], logits[2, 0] = math.nan, math.inf, -math.nan
    tokens = torch.tensor([1, 4999, 3, 4], device="cuda")
    r = appy.token_logprobs(logits, tokens, top=3)
    g = appy.token_logprobs_grad(logits, tokens, r.stats, torch.ones(4, device="cuda"))
    for v in (r.logprobs, r.entropy, r.top_logprobs, g):
        assert v[:3].isnan().all() and v[3].isfinite().all()
    assert ((r.top_tokens >= 0) & (r.top_tokens < 5000)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_top_tokens_wherever_the_large_values_lie(rt, dtype, top):
    cols = 40000
    rising = torch.arange(cols, device="cuda", dtype=torch.float32) / 400
    rows = [rising, rising.flip(0), torch.zeros(cols, device="cuda"), torch.full((cols,), -math.inf, device="cuda"), rising.remainder(7.0)]
    v = 4 if dtype == torch.float32 else 8
    for step in (512 * v, 1024 * v, 4096 * v):          # all of one thread's packs hold the large values
        r = -rising.remainder(1.0) - 50
        for k in range(v):
            r[k::step] = 10 + rising[k::step] % 3
        rows.append(r)
    logits = torch.stack(rows).to(dtype)
    check_logprobs(logits, torch.arange(len(rows), device="cuda") * 17, 1.0, top)
    check_logprobs(torch.cat([logits] * 60), torch.arange(60 * len(rows), device="cuda") * 17, 1.0, top)      # one block per row


def test_token_logprobs_shapes_and_strides(rt):
    base = randn(2, 3, 1100, dtype=torch.bfloat16, seed=1)
    tokens = torch.randint(0, 900, (2, 3), generator=gen(2), device="cuda")
    check_logprobs(base[..., 100:1000], tokens, top=4)                   # rows of a wider array, 16-byte aligned or not
    check_logprobs(base[..., 101:1001], tokens, top=4)
    check_logprobs(base[:, :2, :900], tokens[:, :2], top=4)              # rows not evenly spaced: copied first
    check_logprobs(base[..., :900].transpose(0, 1), tokens.t(), top=4)
    one = appy.token_logprobs(base[0, 0], tokens[0, 0], top=2)
    assert one.logprobs.shape == () and one.top_tokens.shape == (2,) and one.stats.shape == (3,)
    none = appy.token_logprobs(base[:0, 0], tokens[:0, 0], top=2)
    assert none.logprobs.shape == (0,) and none.top_logprobs.shape == (0, 2)


@pytest.mark.parametrize("cols", [1000, 1001, 777])
def test_token_logprobs_grad_in_place_broadcast_and_out(rt, cols):
    logits, tokens = randn(6, cols, dtype=torch.bfloat16, seed=1), torch.randint(0, cols, (6,), generator=gen(2), device="cuda")
    r = appy.token_logprobs(logits, tokens)
    ones = torch.ones((), device="cuda").expand(6)
    ref = appy.token_logprobs_grad(logits, tokens, r.stats, torch.ones(6, device="cuda"), torch.full((6,), 0.5, device="cuda"))
    assert torch.equal(appy.token_logprobs_grad(logits, tokens, r.stats, ones, ones * 0.5), ref)
    assert not appy.token_logprobs_grad(logits, tokens, r.stats).any()   # no gradient comes in, none goes out
    buffer = torch.full((6, cols + 30), 5.0, dtype=torch.bfloat16, device="cuda")
    for at in (0, 8, 11):                                                # rows aligned like the logits', and not
        buffer.fill_(5.0)
        appy.token_logprobs_grad(logits, tokens, r.stats, ones, ones * 0.5, out=buffer[:, at:at + cols])
        assert torch.equal(buffer[:, at:at + cols], ref) and (buffer[:, :at] == 5).all() and (buffer[:, at + cols:] == 5).all()
    own = logits.clone()
    got = appy.token_logprobs_grad(own, tokens, r.stats, ones, ones * 0.5, out=own)
    assert got is own and torch.equal(own, ref)


def test_token_logprobs_gradient_against_differences(rt):
    logits, tokens = randn(3, 11, seed=1), torch.tensor([4, 0, 10], device="cuda")
    g, gh = randn(3, seed=2), randn(3, seed=3)
    r = appy.token_logprobs(logits, tokens, temperature=0.7)
    got = appy.token_logprobs_grad(logits, tokens, r.stats, g, gh, 0.7)

    def loss(x):
        logp = torch.log_softmax(x / 0.7, -1)
        return (g.double() * logp[torch.arange(3), tokens]).sum() - (gh.double()[:, None] * logp.exp() * logp).sum()

    for k in range(33):
        up, down = logits.double(), logits.double()
        up.view(-1)[k] += 1e-6
        down.view(-1)[k] -= 1e-6
        assert abs(float(loss(up) - loss(down)) / 2e-6 - float(got.view(-1)[k])) < 1e-4


# ------------------------------------------------------------------------------------------------ large arrays

def test_offsets_past_32_bits(rt):
    """Arrays of more than 2^31 elements: their last rows agree with calls on those rows alone."""
    rows, width = (1 << 19) + 5, 4104                                     # 2.15e9 elements
    w = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    w[-64:] = randn(64, width, dtype=torch.bfloat16, seed=1)
    w[:64] = 1.0
    tokens = torch.randint(rows - 64, rows, (50,), generator=gen(2), device="cuda")
    assert torch.equal(appy.embedding(w, tokens), w[tokens])
    grad = randn(50, width, dtype=torch.bfloat16, seed=3)
    appy.embedding_grad(grad, tokens, out=w)
    assert torch.equal(w[-64:], appy.embedding_grad(grad, tokens - (rows - 64), 64)) and not w[:64].any() and not w[rows // 2].any()
    tokens = torch.randint(rows - 64, rows, (5000,), generator=gen(4), device="cuda")
    grad = randn(5000, width, dtype=torch.bfloat16, seed=5)
    appy.embedding_grad(grad, tokens, out=w)
    assert torch.equal(w[-64:], appy.embedding_grad(grad, tokens - (rows - 64), 64)) and not w[:64].any()
    del w
    n, cols = 16400, 131072
    logits = torch.zeros(n, cols, dtype=torch.bfloat16, device="cuda")
    logits[-8:] = randn(8, cols, dtype=torch.bfloat16, seed=6)
    tokens = torch.randint(0, cols, (n,), generator=gen(7), device="cuda")
    g = randn(n, seed=8)
    r = appy.token_logprobs(logits, tokens, top=3)
    few = appy.token_logprobs(logits[-8:], tokens[-8:], top=3)
    within(r.logprobs[-8:], few.logprobs.double(), logprob_tolerance(cols) + 8 * U * few.logprobs.double().abs())
    assert torch.equal(r.top_tokens[-8:], few.top_tokens)
    want = appy.token_logprobs_grad(logits[-8:], tokens[-8:], r.stats[-8:], g[-8:])
    appy.token_logprobs_grad(logits, tokens, r.stats, g, out=logits)
    assert torch.equal(logits[-8:], want)
    del logits
    t, d = (1 << 20) + 3, 2056
    x = torch.zeros(1, t, d, dtype=torch.bfloat16, device="cuda")
    x[:, -300:] = randn(1, 300, d, dtype=torch.bfloat16, seed=9)
    h, last = appy.gated_scan(x, x)
    end, last2 = appy.gated_scan(x[:, -300:], x[:, -300:])
    within(last, last2.double(), 1e-5 + 1e-5 * last2.double().abs())
    within(h[:, -300:], end.double(), 2 * half(torch.bfloat16) * end.double().abs() + 1e-5)


# ------------------------------------------------------------------------------------------------ as they are used

def test_refusals(rt):
    w, tokens = randn(10, 8), torch.zeros(4, dtype=torch.int64, device="cuda")
    x = randn(2, 5, 8)
    logits = randn(4, 8)
    for error, call in [
            (TypeError, lambda: appy.embedding(w.double(), tokens)), (TypeError, lambda: appy.embedding(w, tokens.float())),
            (TypeError, lambda: appy.embedding(w, tokens.short())), (ValueError, lambda: appy.embedding(x, tokens)),
            (ValueError, lambda: appy.embedding(w, tokens, out=randn(4, 7))), (ValueError, lambda: appy.embedding(w, tokens, out=randn(4, 8).half())),
            (ValueError, lambda: appy.embedding(w, tokens, out=randn(8, 4).t())), (TypeError, lambda: appy.embedding(w, np.zeros(4, np.int64))),
            (ValueError, lambda: appy.embedding(w, tokens, out=randn(1, 8).expand(4, 8))), (TypeError, lambda: appy.embedding([1.0], tokens)),
            (ValueError, lambda: appy.embedding(w, tokens.cpu())), (ValueError, lambda: appy.gated_scan(x, x, randn(2, 8).cpu())),
            (ValueError, lambda: appy.token_logprobs_grad(logits, tokens, randn(4, 3).cpu())),
            (ValueError, lambda: appy.embedding_grad(randn(4, 8), tokens)), (ValueError, lambda: appy.embedding_grad(randn(3, 8), tokens, 10)),
            (ValueError, lambda: appy.embedding_grad(randn(4, 8), tokens, 10, accumulate=True)),
            (ValueError, lambda: appy.embedding_grad(randn(4, 8), tokens, 10, out=randn(9, 8))),
            (ValueError, lambda: appy.embedding_grad(randn(4, 8), tokens, out=randn(9, 8).half())),
            (ValueError, lambda: appy.gated_scan(x[0], x[0])), (ValueError, lambda: appy.gated_scan(x, x[:, :4])),
            (ValueError, lambda: appy.gated_scan(x, x.half())), (ValueError, lambda: appy.gated_scan(x, x, randn(2, 8).half())),
            (ValueError, lambda: appy.gated_scan(x, x, randn(3, 8))), (ValueError, lambda: appy.gated_scan(x, x, offsets=tokens)),
            (TypeError, lambda: appy.gated_scan(x[0], x[0], offsets=tokens.float())), (ValueError, lambda: appy.gated_scan(x[0], x[0], offsets=tokens[:0])),
            (ValueError, lambda: appy.gated_scan(x, x, out=randn(2, 5, 1).expand(2, 5, 8))),
            (ValueError, lambda: appy.gated_scan(x, x, out=randn(1, 5, 8).expand(2, 5, 8))),
            (ValueError, lambda: appy.gated_scan(x, x, last=randn(8, 2).t())), (ValueError, lambda: appy.gated_scan_grad(x, x, x, x.half())),
            (ValueError, lambda: appy.gated_scan_grad(x[:1], x, x, x)), (ValueError, lambda: appy.gated_scan_grad(x, x, x, x, out=(x, x.half()))),
            (ValueError, lambda: appy.token_logprobs(logits, tokens[:3])), (ValueError, lambda: appy.token_logprobs(logits, tokens, top=9)),
            (ValueError, lambda: appy.token_logprobs(logits[:, :0], tokens)), (TypeError, lambda: appy.token_logprobs(logits.int(), tokens)),
            (RuntimeError, lambda: appy.token_logprobs(logits, tokens, temperature=0.0)),
            (ValueError, lambda: appy.token_logprobs_grad(logits, tokens, randn(4, 2))),
            (ValueError, lambda: appy.token_logprobs_grad(logits, tokens, randn(4, 3), randn(4).half())),
            (ValueError, lambda: appy.token_logprobs_grad(logits, tokens, randn(4, 3), randn(3))),
            (RuntimeError, lambda: appy.embedding(w.clone().requires_grad_(), tokens)),
            (RuntimeError, lambda: appy.gated_scan(x, x.clone().requires_grad_())),
            (RuntimeError, lambda: appy.token_logprobs(logits.clone().requires_grad_(), tokens))]:
        before = rt.launch_count()
        with pytest.raises(error):
            call()
        assert rt.launch_count() == before
    with torch.no_grad():
        appy.embedding(w.clone().requires_grad_(), tokens)


def test_host_arrays(rt):
    rng = np.random.default_rng(0)
    w, tokens = rng.standard_normal((20, 12), dtype=np.float32), rng.integers(0, 20, (3, 4))
    e = appy.embedding(w, tokens)
    assert isinstance(e, np.ndarray) and np.array_equal(e, w[tokens])
    out = np.empty((3, 4, 12), np.float32)
    assert appy.embedding(w, tokens, out=out) is out and np.array_equal(out, e)
    dw = np.ones((20, 12), np.float32)
    appy.embedding_grad(e, tokens, out=dw, accumulate=True)
    ref = np.ones((20, 12))
    np.add.at(ref, tokens.reshape(-1), e.reshape(-1, 12).astype(np.float64))
    assert np.allclose(dw, ref, rtol=1e-5, atol=1e-5)
    h, last = appy.gated_scan(e, e[::-1].copy())
    dev = torch.from_numpy(e).cuda()
    h2, last2 = appy.gated_scan(dev, dev.flip(0))
    assert isinstance(last, np.ndarray) and np.array_equal(h, h2.cpu().numpy()) and np.array_equal(last, last2.cpu().numpy())
    dx, dg, d0 = appy.gated_scan_grad(e, e, e[::-1].copy(), h)
    assert np.array_equal(dg, appy.gated_scan_grad(dev, dev, dev.flip(0), h2)[1].cpu().numpy())
    cpu = torch.from_numpy(w)
    r = appy.token_logprobs(cpu, torch.arange(12).repeat(2)[:20], top=3)
    assert r.top_tokens.device.type == "cpu" and torch.equal(r.top_tokens[:, 0], cpu.argmax(1))
    g = appy.token_logprobs_grad(cpu, torch.arange(12).repeat(2)[:20], r.stats, torch.ones(20))
    assert g.device.type == "cpu" and g.sum(1).abs().max() < 1e-5


def test_inside_a_jitted_function_beside_a_loop(rt):
    w, tokens = randn(30, 40, seed=1), torch.randint(0, 30, (25,), generator=gen(2), device="cuda")
    got = jitted_mix(w, tokens, torch.empty(25, 40, device="cuda"))
    assert torch.equal(got, appy.embedding(w, tokens) * 2 + 1)


@appy.jit
def jitted_mix(w, tokens, out):
    e = appy.embedding(w, tokens)
    #pragma parallel for
    for i in range(out.shape[0]):
        #pragma simd
        for j in range(out.shape[1]):
            out[i, j] = e[i, j] * 2.0 + 1.0
    return out


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens):
        ctx.save_for_backward(tokens)
        ctx.rows = weight.shape[0]
        return appy.embedding(weight, tokens, scale=1.5)

    @staticmethod
    def backward(ctx, grad):
        return appy.embedding_grad(grad, ctx.saved_tensors[0], ctx.rows, scale=1.5), None


class Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate):
        h, _ = appy.gated_scan(x, gate)
        ctx.save_for_backward(x, gate, h)
        return h

    @staticmethod
    def backward(ctx, grad):
        return appy.gated_scan_grad(grad, *ctx.saved_tensors)[:2]


class TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens):
        r = appy.token_logprobs(logits, tokens)
        ctx.save_for_backward(logits, tokens, r.stats)
        return r.logprobs, r.entropy

    @staticmethod
    def backward(ctx, g, gh):
        return appy.token_logprobs_grad(*ctx.saved_tensors, g, gh), None


def test_a_recurrent_language_model_trains(rt):
    """Tokens -> embedding -> gated recurrence -> logits -> log probabilities, and the gradients of every weight against
    the same model in float64.  All of it is float32 with sums of at most a few hundred terms of order one: 1e-4 of a
    gradient's largest value is some hundred roundings."""
    b, t, d, v = 3, 70, 48, 211
    tokens = torch.randint(0, v, (b, t + 1), generator=gen(1), device="cuda")
    weights = [randn(v, d, seed=2), randn(d, 2 * d, seed=3, std=0.2), randn(d, v, seed=4, std=0.3)]
    tokens[0, 50:] = -100                                                # a padded batch

    def run(ws, embed, scan, logprobs):
        e = embed(ws[0], tokens[:, :-1])
        p = e @ ws[1]
        h = scan(p[..., :d], p[..., d:])
        lp, entropy = logprobs(h @ ws[2], tokens[:, 1:])
        return -lp.sum() - 0.1 * (entropy * (tokens[:, 1:] >= 0)).sum()

    def embed64(w, t):
        return torch.where((t >= 0)[..., None], w[t.clamp_min(0)] * 1.5, 0.0)

    def scan64(x, gate):
        s, out = torch.zeros_like(x[:, 0]), []
        for k in range(x.shape[1]):
            f = torch.sigmoid(gate[:, k])
            s = f * s + (1 - f) * x[:, k]
            out.append(s)
        return torch.stack(out, 1)

    def logprobs64(z, t):
        logp = torch.log_softmax(z, -1)
        return torch.where(t >= 0, logp.gather(-1, t.clamp_min(0)[..., None])[..., 0], 0.0), -(logp.exp() * logp).sum(-1)

    mine = [w.clone().requires_grad_() for w in weights]
    ref = [w.double().requires_grad_() for w in weights]
    loss = run(mine, Embedding.apply, Scan.apply, TokenLogprobs.apply)
    loss64 = run(ref, embed64, scan64, logprobs64)
    loss.backward()
    loss64.backward()
    assert abs(float(loss.detach()) - float(loss64.detach())) < 1e-4 * abs(float(loss64.detach()))
    for a, r in zip(mine, ref):
        assert (a.grad.double() - r.grad).abs().max() < 1e-4 * r.grad.abs().max()


def step(w, tokens, x, gate, logits, g):
    e = appy.embedding(w, tokens)
    dw = appy.embedding_grad(e, tokens, w.shape[0])
    h, last = appy.gated_scan(x, gate)
    dx, dg, d0 = appy.gated_scan_grad(x, x, gate, h, grad_last=last)
    r = appy.token_logprobs(logits, tokens, top=5)
    dl = appy.token_logprobs_grad(logits, tokens, r.stats, g, g)
    return e, dw, h, last, dx, dg, d0, r.logprobs, r.entropy, r.top_logprobs, r.top_tokens, dl


def step_inputs(seed):
    return (randn(3000, 64, dtype=torch.bfloat16, seed=seed), torch.randint(-1, 3000, (5000,), generator=gen(seed), device="cuda"),
            randn(1, 3000, 128, dtype=torch.bfloat16, seed=seed + 1), randn(1, 3000, 128, dtype=torch.bfloat16, seed=seed + 2),
            randn(5000, 3000, dtype=torch.bfloat16, seed=seed + 3), randn(5000, seed=seed + 4))


def test_captured_and_replayed(rt):
    a, b = step_inputs(1), step_inputs(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for inputs in (a, b):
            step(*inputs)
    torch.cuda.synchronize()
    for inputs in (a, b):                                # two graphs of the same stream, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(*inputs)
        graphs.append((graph, out, inputs))
    new = step_inputs(7)
    for k, (graph, out, inputs) in enumerate(graphs):
        for mine, other in zip(inputs, new if k else a):
            mine.copy_(other)
    expect = [[v.clone() for v in step(*inputs)] for _, _, inputs in graphs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out, _), want in zip(graphs, expect):
        for got, ref in zip(out, want):
            assert torch.equal(got.nan_to_num(), ref.nan_to_num())


def test_two_streams_at_once(rt):
    inputs = [step_inputs(1), step_inputs(2)]
    expect = [[v.clone() for v in step(*i)] for i in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = step(*inputs[k])
    torch.cuda.synchronize()
    for g, e in zip(got, expect):
        for x, y in zip(g, e):
            assert torch.equal(x, y)
