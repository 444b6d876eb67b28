"""The C entries of the language-model operators refuse bad arguments before any launch (no GPU needed)."""
import ctypes as C

import pytest

from appy_b200.backends.cuda_sm100 import runtime as rt

F32, F64, I32, I64, F16, BF16 = range(6)
P = C.c_void_p(4096)          # stands for a device pointer; nothing here gets as far as using it
N = None


def refused(name, *args):
    status = getattr(rt.lib(), name)(*args, None)
    assert status == -3
    message = rt.lib().appy_last_error().decode()
    assert message.startswith(name + ":")
    return message


def embedding(w=P, dtype=F32, ldw=8, rows=10, width=8, tokens=P, token_dtype=I64, n=4, out=P, ldo=8):
    return "appy_embedding", w, dtype, ldw, rows, width, tokens, token_dtype, n, 1.0, out, ldo


@pytest.mark.parametrize("bad, word", [
    (dict(dtype=F64), "dtype"), (dict(dtype=I32), "dtype"), (dict(dtype=-1), "dtype"), (dict(token_dtype=F32), "token_dtype"),
    (dict(rows=-1), "negative"), (dict(n=-1), "negative"), (dict(width=-8), "negative"), (dict(w=N), "NULL"), (dict(tokens=N), "NULL"),
    (dict(out=N), "NULL"), (dict(ldw=7), "ldw"), (dict(ldo=7), "ldo"), (dict(width=1 << 31, ldw=1 << 31, ldo=1 << 31), "width"),
    (dict(n=1 << 50), "too many")])
def test_embedding(bad, word):
    assert word in refused(*embedding(**bad))


def grad(g=P, dtype=F32, ldg=8, tokens=P, token_dtype=I32, n=4, rows=10, width=8, out=P, out_dtype=F32, ldo=8, ws=P, size=1 << 30):
    return "appy_embedding_grad", g, dtype, ldg, tokens, token_dtype, n, rows, width, 1.0, 0, out, out_dtype, ldo, ws, size


@pytest.mark.parametrize("bad, word", [
    (dict(dtype=I64), "dtype"), (dict(dtype=F16, out_dtype=BF16), "out_dtype"), (dict(out_dtype=F16), "out_dtype"),
    (dict(token_dtype=BF16), "token_dtype"), (dict(n=1 << 31), "sizes"), (dict(rows=1 << 31), "sizes"), (dict(n=-1), "sizes"),
    (dict(g=N), "NULL"), (dict(tokens=N), "NULL"), (dict(out=N), "NULL"), (dict(ws=N), "NULL"), (dict(ldg=7), "ldg"), (dict(ldo=3), "ldo"),
    (dict(size=255), "workspace"), (dict(ws=C.c_void_p(4096 + 64)), "workspace")])
def test_embedding_grad(bad, word):
    assert word in refused(*grad(**bad))


def test_embedding_grad_workspace_size():
    size = C.c_size_t()
    assert rt.lib().appy_embedding_grad_bytes(0, 0, 0, C.byref(size)) == 0 and size.value > 0
    small = size.value
    assert rt.lib().appy_embedding_grad_bytes(1 << 20, 1 << 17, 4096, C.byref(size)) == 0 and size.value > small
    assert rt.lib().appy_embedding_grad_bytes(1 << 31, 10, 8, C.byref(size)) == -3
    assert rt.lib().appy_embedding_grad_bytes(10, 10, 8, None) == -3


def scan(x=P, gate=P, dtype=BF16, offsets=N, offsets_dtype=I32, sequences=2, tokens=5, width=8, h=P):
    return "appy_gated_scan", x, 40, 8, gate, 40, 8, dtype, offsets, offsets_dtype, sequences, tokens, width, N, h, 40, 8, P, 0


def scan_grad(dh=P, x=P, gate=P, h=P, dtype=BF16, offsets=N, offsets_dtype=I32, sequences=2, tokens=5, width=8, gx=P, gg=P):
    return ("appy_gated_scan_grad", dh, 40, 8, x, 40, 8, gate, 40, 8, h, 40, 8, dtype, offsets, offsets_dtype, sequences, tokens, width, N, N,
            gx, 40, 8, gg, 40, 8, P, 0)


BAD_SCAN = [(dict(dtype=F64), "dtype"), (dict(offsets=P, offsets_dtype=F32), "offsets_dtype"), (dict(sequences=-1), "negative"),
            (dict(tokens=-1), "negative"), (dict(width=-1), "negative"), (dict(width=1 << 31), "width"), (dict(x=N), "NULL"),
            (dict(gate=N), "NULL"), (dict(h=N), "NULL"), (dict(sequences=1 << 40), "too many")]


@pytest.mark.parametrize("bad, word", BAD_SCAN)
def test_gated_scan(bad, word):
    assert word in refused(*scan(**bad))


@pytest.mark.parametrize("bad, word", BAD_SCAN + [(dict(gx=N), "NULL"), (dict(gg=N), "NULL")])
def test_gated_scan_grad(bad, word):
    assert word in refused(*scan_grad(**bad))


def logprobs(x=P, dtype=F32, ld=100, rows=4, cols=100, tokens=P, token_dtype=I64, temperature=1.0, top=0, lp=P, h=P, stats=P, tv=N, ti=N):
    return "appy_token_logprobs", x, dtype, ld, rows, cols, tokens, token_dtype, temperature, top, lp, h, stats, tv, ti


def logprobs_grad(x=P, dtype=F32, ld=100, rows=4, cols=100, tokens=P, token_dtype=I64, temperature=1.0, stats=P, out=P, ldo=100):
    return "appy_token_logprobs_grad", x, dtype, ld, rows, cols, tokens, token_dtype, temperature, stats, N, 1, N, 1, out, ldo


BAD_ROWS = [(dict(dtype=I32), "dtype"), (dict(token_dtype=F16), "token_dtype"), (dict(rows=-1), "rows"), (dict(cols=0), "cols"),
            (dict(cols=1 << 31, ld=1 << 31), "cols"), (dict(ld=99), "ld"), (dict(temperature=0.0), "temperature"),
            (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
            (dict(temperature=float("inf")), "temperature"), (dict(x=N), "NULL"), (dict(tokens=N), "NULL"), (dict(stats=N), "NULL"),
            (dict(rows=1 << 40), "too many")]


@pytest.mark.parametrize("bad, word", BAD_ROWS + [(dict(top=-1), "top"), (dict(top=33), "top"), (dict(top=11, cols=10), "top"), (dict(top=2), "NULL"),
                                                  (dict(lp=N), "NULL"), (dict(h=N), "NULL")])
def test_token_logprobs(bad, word):
    assert word in refused(*logprobs(**bad))


@pytest.mark.parametrize("bad, word", BAD_ROWS + [(dict(out=N), "NULL"), (dict(ldo=99), "ldo")])
def test_token_logprobs_grad(bad, word):
    assert word in refused(*logprobs_grad(**bad))


def test_nothing_to_do_is_no_error():
    lib = rt.lib()
    for name, *args in (embedding(n=0, tokens=N, out=N), embedding(width=0), grad(rows=0), grad(width=0), scan(sequences=0), scan(width=0),
                        scan_grad(sequences=0), logprobs(rows=0), logprobs_grad(rows=0)):
        assert getattr(lib, name)(*args, None) == 0


@pytest.mark.parametrize("n", [(1 << 31) - 2, (1 << 31) - 1024, (1 << 31) - (1 << 16) + 1])
def test_embedding_grad_of_positions_whose_shares_would_pass_32_bits(n):
    size = C.c_size_t()
    assert "sizes" in refused(*grad(n=n, size=1 << 40))
    assert rt.lib().appy_embedding_grad_bytes(n, 10, 8, C.byref(size)) == -3
    assert rt.lib().appy_embedding_grad_bytes((1 << 31) - (1 << 16), 10, 8, C.byref(size)) == 0
