"""The language-model operators at the edges of what they accept: values, aliases and callers that ordinary use does not reach."""
import math

import numpy as np
import pytest

import appy_b200 as appy

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_operators_gpu import TYPES, U, TokenLogprobs, check_logprobs, gen, grad_reference, grad_tolerance, randn, within  # noqa: E402


# ------------------------------------------------------------------------------------------------ log probabilities

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -1e30, -1e37])
@pytest.mark.parametrize("temperature", [0.5, 0.6, 0.7, 0.8, 1.0, 2.0])
def test_token_logprobs_masked_by_large_finite_values(rt, dtype, mask, temperature):
    """Every distance from a logit to the row's maximum is taken from the maximum itself where the product of the maximum
    and log2(e) / temperature would be rounded by more than a fraction of one: the bounds are those of any other row."""
    for cols in (37, 3001, 20000):
        wide = randn(9, cols + 1, dtype=dtype, seed=cols, std=2.0)
        for logits in (wide[:, :cols], wide[:, 1:]):             # rows on 16 bytes or not, and all off them
            logits[0] = mask                                     # nothing else
            logits[1, cols // 2:] = mask                         # a padded vocabulary's tail
            logits[2, : cols // 2] = mask
            logits[3] = mask
            logits[3, cols // 3] = 1.5                           # one left
            logits[4, 0] = mask
            logits[5, ::2] = mask
            logits[6] = -mask                                    # large and positive
            logits[7, cols - 1] = -mask
            logits[8] = mask
            logits[8, 0] = 2 * mask                              # two kinds
            logits[8, cols - 1] = mask * 0.75
            tokens = torch.randint(0, cols, (9,), generator=gen(2), device="cuda")
            tokens[1], tokens[2], tokens[3] = 3, cols - 1, cols // 3
            check_logprobs(logits, tokens, temperature, min(20, cols))
    check_logprobs(torch.cat([logits] * 40), torch.cat([tokens] * 40), temperature, 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-4, 1e4])
@pytest.mark.parametrize("std", [1.0, 100.0, 1e4])
def test_token_logprobs_at_both_ends_of_the_temperature(rt, dtype, temperature, std):
    for cols in (9, 1001, 20000):
        logits = randn(5, cols, dtype=dtype, seed=cols, std=std)
        logits[1] += 3 * std
        logits[2] -= 3 * std
        logits[3, ::3] = -math.inf
        tokens = logits.argmax(-1)
        tokens[4] = cols - 1
        check_logprobs(logits, tokens, temperature, 5)


def test_results_of_log_probabilities_are_arrays_of_their_own(rt):
    logits, tokens = randn(6, 50, seed=1).requires_grad_(), torch.arange(6, device="cuda")
    lp, entropy = TokenLogprobs.apply(logits, tokens)
    keep = (tokens % 2 == 0).float()
    lp.mul_(keep)                                                # in place, as a loss over a padded batch does it
    entropy.masked_fill_(keep == 0, 0.0)
    (lp.sum() + entropy.sum()).backward()
    r = appy.token_logprobs(logits.detach(), tokens, top=3)
    assert torch.equal(logits.grad, appy.token_logprobs_grad(logits.detach(), tokens, r.stats, keep, keep))
    stats = r.stats.clone()
    before = r.stats._version
    r.logprobs.zero_(), r.entropy.zero_(), r.top_logprobs.zero_()
    assert torch.equal(r.stats, stats) and r.stats._version == before
    for v in r:
        assert not v._is_view() and v.untyped_storage().nbytes() == v.numel() * v.element_size()


# ------------------------------------------------------------------------------------------------ autograd

def test_forward_mode_is_refused(rt):
    import torch.autograd.forward_ad as fwad
    w, tokens, x, logits = randn(10, 8, seed=1), torch.arange(4, device="cuda"), randn(2, 5, 8, seed=2), randn(4, 8, seed=3)
    h, _ = appy.gated_scan(x, x)
    stats = appy.token_logprobs(logits, tokens).stats
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in [lambda: appy.embedding(dual(w), tokens), lambda: appy.embedding_grad(dual(logits), tokens, 10), lambda: appy.gated_scan(x, dual(x)),
                     lambda: appy.gated_scan(x, x, dual(x[:, 0].contiguous())), lambda: appy.gated_scan_grad(dual(x), x, x, h),
                     lambda: appy.token_logprobs(dual(logits), tokens), lambda: appy.token_logprobs_grad(dual(logits), tokens, stats),
                     lambda: appy.embedding(dual(w.cpu()), tokens.cpu())]:
            before = rt.launch_count()
            with pytest.raises(RuntimeError, match="autograd"):
                call()
            assert rt.launch_count() == before
        assert torch.equal(appy.embedding(w, tokens), w[tokens])         # without a tangent it goes on as ever


# ------------------------------------------------------------------------------------------------ embedding

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [8, 100, 769, 1024])
@pytest.mark.parametrize("scale", [-2.0, math.inf, -math.inf, math.nan])
def test_unknown_tokens_give_positive_zeros_whatever_the_scale(rt, dtype, width, scale):
    w = randn(20, width, dtype=dtype, seed=1)
    tokens = torch.tensor([-1, 3, 20, 7, 1 << 40, -(1 << 40)], device="cuda")
    got = appy.embedding(w, tokens, scale=scale)
    unknown = got[[0, 2, 4, 5]]
    assert not unknown.any() and not torch.signbit(unknown).any()
    assert torch.equal(got[[1, 3]].nan_to_num(7.0), (w[[3, 7]].float() * scale).to(dtype).nan_to_num(7.0))


@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("width", [8, 7])
def test_embedding_grad_accumulates_subnormal_values(rt, n, width):
    small = 2.0 ** -140
    out = torch.full((4, width), small, device="cuda")
    tokens = torch.full((n,), 2, device="cuda")
    grad = torch.zeros(n, width, device="cuda")
    appy.embedding_grad(grad, tokens, out=out, accumulate=True)
    assert (out == small).all()                                  # zeros added
    grad[0] = 3 * small
    appy.embedding_grad(grad, tokens, out=out, accumulate=True)
    assert (out[2] == 4 * small).all() and (out[[0, 1, 3]] == small).all()


@pytest.mark.parametrize("n", [200, 700])
@pytest.mark.parametrize("width", [64, 61])
def test_embedding_grad_accumulates_with_one_rounding_down_to_the_smallest_values(rt, n, width):
    """Every row has one position: the result is the sum of two float32 numbers, rounded once."""
    gradient = torch.randn(n, width, generator=gen(1), device="cuda") * 2.0 ** torch.randint(-149, -99, (n, width), generator=gen(2), device="cuda").double()
    old = torch.randn(n, width, generator=gen(3), device="cuda") * 2.0 ** torch.randint(-149, -99, (n, width), generator=gen(4), device="cuda").double()
    gradient, old = gradient.float(), old.float()
    old[:, ::5] = -gradient[:, ::5] * (1 + 2.0 ** -20)           # nearly cancelling
    gradient[: n // 2] = torch.where(gradient[: n // 2].abs() < 2.0 ** -101, 2.0 ** -101, gradient[: n // 2])      # the other way of adding
    tokens = torch.randperm(n, generator=gen(5), device="cuda")
    out = old.clone()
    appy.embedding_grad(gradient, tokens, out=out, accumulate=True)
    want = (old[tokens].double() + gradient.double()).float()    # 2^-149 to 2^-96: exact in 64 bits, then rounded
    assert torch.equal(out[tokens], want)


@pytest.mark.parametrize("dtype, out_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.float32),
                                              (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("n", [40, 256, 257, 3000])
@pytest.mark.parametrize("width", [64, 67, 1])
def test_embedding_grad_accumulates_in_every_form(rt, dtype, out_dtype, n, width):
    rows = 90
    tokens = torch.randint(-2, rows + 2, (n,), generator=gen(n), device="cuda")
    tokens[: n // 3] = 5                                         # one frequent row
    grad, out = randn(n, width, dtype=dtype, seed=1), randn(rows, width, dtype=out_dtype, seed=2)
    before = out.clone()
    got = appy.embedding_grad(grad, tokens, scale=-0.5, out=out, accumulate=True)
    ref, size, count = grad_reference(grad, tokens, rows, -0.5)
    assert got is out
    within(out, ref + before.double(), grad_tolerance(ref + before.double(), size + before.double().abs(), count + 1, out_dtype))
    assert torch.equal(out[count[:, 0] == 0], before[count[:, 0] == 0])


# ------------------------------------------------------------------------------------------------ gated recurrence

@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_sequence_are_cleared_for_no_sequences_too(rt, dtype):
    x = randn(9, 24, dtype=dtype, seed=1)
    out = [torch.full((9, 40), 7.0, dtype=dtype, device="cuda") for _ in range(3)]
    offsets = torch.zeros(1, dtype=torch.int32, device="cuda")
    code = {torch.float32: 0, torch.float16: 4, torch.bfloat16: 5}[dtype]
    stream = torch.cuda.current_stream().cuda_stream

    def place(t):
        return t.data_ptr(), 0, t.stride(0)

    def call(fill):
        rt.check(rt.lib().appy_gated_scan(*place(x), *place(x), code, offsets.data_ptr(), 2, 0, 9, 24, None, *place(out[0]), None, fill, stream))
        rt.check(rt.lib().appy_gated_scan_grad(*place(x), *place(x), *place(x), *place(x), code, offsets.data_ptr(), 2, 0, 9, 24, None, None,
                                               *place(out[1]), *place(out[2]), None, fill, stream))

    call(0)
    assert all((o == 7).all() for o in out)
    call(1)
    assert all(not o[:, :24].any() and (o[:, 24:] == 7).all() for o in out)
    h, last = appy.gated_scan(x, x, offsets=offsets)
    dx, dg, d0 = appy.gated_scan_grad(x, x, x, h, offsets=offsets)
    assert not h.any() and not dx.any() and not dg.any() and last.shape == d0.shape == (0, 24)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("width", [64, 61])
def test_small_gates_and_small_complements_are_exact_to_their_size(rt, packed, width):
    """h = f for x = 0 and a state of one, h = 1 - f for x = 1 and no state; the same factors lead to the gradients of the
    state and of x.  The exponent is rounded once, relative to its size: (1.3 |gate| + 8) 2^-24."""
    at = torch.tensor([0.0, 0.5, -0.5, 5.0, -5.0, 20.0, -20.0, 50.0, -50.0, 80.0, -80.0, 87.0, -87.0, 60.3, -60.3, 33.3], device="cuda")
    gate = at[:, None, None].expand(-1, 1, width).contiguous()
    one, f, i = torch.ones_like(gate), torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    bound = (1.3 * gate.double().abs() + 8) * U
    state = torch.ones(len(at), width, device="cuda")
    offsets, shape = (torch.arange(len(at) + 1, device="cuda"), (len(at), width)) if packed else (None, gate.shape)
    gate, one = gate.view(shape), one.view(shape)
    h, last = appy.gated_scan(torch.zeros_like(one), gate, state, offsets)
    within(h.view(f.shape), f, bound * f)
    assert torch.equal(last, h.view(last.shape))
    h, _ = appy.gated_scan(one, gate, None, offsets)
    within(h.view(i.shape), i, bound * i)
    dx, _, d0 = appy.gated_scan_grad(one, one, gate, h, state, offsets)
    within(dx.view(i.shape), i, bound * i)
    within(d0.view(f.shape), f, bound * f)
    open_, _ = appy.gated_scan(one, torch.full_like(gate, 87.5), None, offsets)
    closed, _ = appy.gated_scan(torch.zeros_like(one), torch.full_like(gate, -100.0), state, offsets)
    assert not open_.any() and ((closed > 1.6e-38) & (closed < 1.7e-38)).all()


# ------------------------------------------------------------------------------------------------ host arrays

@appy.jit
def doubled(a, out):
    #pragma parallel for
    for i in range(out.shape[0]):
        #pragma simd
        for j in range(out.shape[1]):
            out[i, j] = a[i, j] * 2.0
    return out


def test_loops_see_what_an_operator_wrote_to_a_resident_array(rt):
    rng = np.random.default_rng(0)
    w, tokens = rng.standard_normal((20, 12), dtype=np.float32), rng.integers(0, 20, 30)
    whole = np.ones((40, 12), np.float32)
    appy.resident(whole)
    try:
        out = np.empty_like(whole)
        doubled(whole, out)
        assert np.array_equal(out, 2 * whole)
        appy.embedding(w, tokens, out=whole[5:35])               # rows inside it
        assert np.array_equal(whole[5:35], w[tokens])
        doubled(whole, out)
        assert np.array_equal(out, 2 * whole)
        appy.embedding(torch.from_numpy(w), torch.from_numpy(tokens), out=torch.from_numpy(whole)[:30])      # its memory under another name
        doubled(whole, out)
        assert np.array_equal(out, 2 * whole) and np.array_equal(whole[:30], w[tokens])
    finally:
        appy.release(whole)


def test_host_scalars_keep_their_shape(rt):
    w = np.arange(24, dtype=np.float32).reshape(6, 4)
    e = appy.embedding(w, np.array(3))
    assert e.shape == (4,) and np.array_equal(e, w[3])
    r = appy.token_logprobs(w[2], np.array(1), top=2)
    assert r.logprobs.shape == () and r.stats.shape == (3,) and r.top_tokens.shape == (2,)
    assert appy.token_logprobs_grad(w[2], np.array(1), r.stats, r.logprobs).shape == (4,)
    g = appy.embedding_grad(w[0], np.array(2), 5)
    assert g.shape == (5, 4) and np.array_equal(g[2], w[0]) and not g[[0, 1, 3, 4]].any()


def test_a_device_array_given_for_the_results_of_host_arrays_is_returned(rt):
    w = np.arange(24, dtype=np.float32).reshape(6, 4)
    out = torch.empty(2, 4, device="cuda")
    assert appy.embedding(w, np.array([5, 0]), out=out) is out and np.array_equal(out.cpu().numpy(), w[[5, 0]])
    x = w.reshape(2, 3, 4)
    last = torch.empty(2, 4, device="cuda")
    h, got = appy.gated_scan(x, x, last=last)
    assert got is last and isinstance(h, np.ndarray)


def test_read_only_host_arrays_are_not_written(rt):
    w = np.arange(24, dtype=np.float32).reshape(6, 4)
    out = np.zeros((2, 4), np.float32)
    out.flags.writeable = False
    before = rt.launch_count()
    with pytest.raises(ValueError, match="read-only"):
        appy.embedding(w, np.array([5, 0]), out=out)
    assert rt.launch_count() == before and not out.any()
    back = np.zeros((2, 4), np.float32)
    assert appy.embedding(w, np.array([5, 0]), out=back[::-1]) is not None and np.array_equal(back, w[[0, 5]])
