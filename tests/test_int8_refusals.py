"""The 8-bit rows, their product and the log probabilities on a machine without a
GPU: every malformed argument is refused before any device work."""
import ctypes

import pytest

from cq35 import _lib

BASE = 1 << 20  # an address of the right alignment that is never read
BF16, F32 = 0, 1


def lib():
    return _lib.load()


def rows(data=BASE, stride=64, dtype=BF16):
    return _lib.Rows(data, stride, dtype)


def int8(data=BASE, stride=64, scale=BASE):
    return _lib.Int8Rows(data, stride, scale)


def refused(rc, code, text):
    assert rc == code, (rc, lib().cq35_last_error())
    assert text in lib().cq35_last_error().decode(), lib().cq35_last_error()


def ref(x):
    return None if x is None else ctypes.byref(x)


def quantize(x=rows(), n=3, channels=64, out=int8()):
    return lib().cq35_quantize_rows(ref(x), n, channels, ref(out), None)


def norm(x=rows(), residual=rows(), weight=BASE, eps=1e-6, n=3, channels=64, summed=rows(), out=int8()):
    return lib().cq35_norm_quantize(ref(x), ref(residual), weight, eps, n, channels, ref(summed), ref(out), None)


def gated(x=rows(), up=rows(), n=3, channels=64, out=int8()):
    return lib().cq35_gated_quantize(ref(x), ref(up), n, channels, ref(out), None)


def linear(x=int8(), w=int8(), n=3, outputs=64, channels=64, out=rows()):
    return lib().cq35_int8_linear(ref(x), ref(w), n, outputs, channels, ref(out), None)


def logprobs(x=rows(), n=3, vocab=64, tokens=BASE, given=1, top=2, lp=BASE, entropy=BASE, top_tokens=BASE, top_lp=BASE, workspace=BASE,
             size=1 << 40):
    return lib().cq35_token_logprobs(ref(x), n, vocab, tokens, given, top, lp, entropy, top_tokens, top_lp, workspace, size, None)


BAD_ROWS = [
    (None, -1, "null"), (rows(None), -1, "null"), (rows(BASE + 8), -1, "16-byte"), (rows(dtype=2), -4, "type 2"), (rows(dtype=-1), -4, "type -1"),
    (rows(stride=-64), -1, "apart"), (rows(stride=68), -1, "multiple of 8"), (rows(stride=66, dtype=F32), -1, "multiple of 4"),
]
BAD_OUT = [
    (None, -1, "null"), (int8(None), -1, "null"), (int8(scale=None), -1, "null"), (int8(BASE + 4), -1, "16-byte"), (int8(stride=72), -1, "multiple of 16"),
    (int8(stride=-64), -1, "apart"), (int8(stride=48), -1, "overlap"), (int8(stride=0), -1, "overlap"),
]


@pytest.mark.parametrize("call", [quantize, norm, gated])
@pytest.mark.parametrize("bad,code,text", BAD_ROWS)
def test_input_refusals(call, bad, code, text):
    refused(call(x=bad), code, text)


@pytest.mark.parametrize("call", [quantize, norm, gated])
@pytest.mark.parametrize("bad,code,text", BAD_OUT)
def test_output_refusals(call, bad, code, text):
    refused(call(out=bad), code, text)


@pytest.mark.parametrize("call", [quantize, norm, gated, linear])
@pytest.mark.parametrize("change,code,text", [
    (dict(n=-1), -2, "rows"), (dict(n=(1 << 21) + 1), -2, "rows"), (dict(channels=0), -2, "channels"), (dict(channels=24), -2, "channels"),
    (dict(channels=-16), -2, "channels"), (dict(channels=65552), -2, "channels"),
])
def test_size_refusals(call, change, code, text):
    refused(call(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(weight=None), -1, "null"), (dict(weight=BASE + 8), -1, "16-byte"), (dict(eps=-1e-6), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(residual=rows(BASE + 2)), -1, "16-byte"), (dict(residual=rows(dtype=F32)), -1, "types"), (dict(summed=None), -1, "null"),
    (dict(summed=rows(stride=32)), -1, "overlap"), (dict(summed=rows(dtype=F32)), -1, "types"),
])
def test_norm_refusals(change, code, text):
    refused(norm(**change), code, text)


@pytest.mark.parametrize("change,code,text", [(dict(up=None), -1, "null"), (dict(up=rows(dtype=F32)), -1, "types"), (dict(up=rows(stride=4)), -1, "multiple")])
def test_gated_refusals(change, code, text):
    refused(gated(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), -1, "null"), (dict(x=int8(scale=None)), -1, "null"), (dict(w=int8(None)), -1, "null"), (dict(w=int8(BASE + 8)), -1, "16-byte"),
    (dict(x=int8(stride=40)), -1, "multiple of 16"), (dict(outputs=0), -2, "outputs"), (dict(outputs=-5), -2, "outputs"),
    (dict(outputs=(1 << 21) + 1), -2, "outputs"), (dict(n=1 << 21, outputs=1 << 21, out=rows(stride=1 << 21)), -2, "too many"), (dict(out=None), -1, "null"),
    (dict(out=rows(None)), -1, "null"), (dict(out=rows(dtype=7)), -4, "type 7"), (dict(out=rows(BASE + 1)), -1, "misaligned"),
    (dict(out=rows(BASE + 2, dtype=F32)), -1, "misaligned"), (dict(out=rows(stride=63)), -1, "overlap"), (dict(out=rows(stride=-64)), -1, "overlap"),
])
def test_linear_refusals(change, code, text):
    refused(linear(**change), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(n=-1), -2, "rows"), (dict(n=(1 << 21) + 1), -2, "rows"), (dict(vocab=0), -2, "logits"), (dict(vocab=(1 << 30) + 1), -2, "logits"),
    (dict(given=-1), -2, "given"), (dict(given=1025), -2, "given"), (dict(top=-1), -2, "alternatives"), (dict(top=33), -2, "alternatives"),
    (dict(vocab=5, top=6), -2, "alternatives"), (dict(x=None), -1, "null"), (dict(x=rows(None)), -1, "null"), (dict(x=rows(dtype=2)), -4, "type 2"),
    (dict(x=rows(BASE + 1)), -1, "misaligned"), (dict(x=rows(BASE + 2, dtype=F32)), -1, "misaligned"), (dict(x=rows(stride=-1)), -1, "apart"),
    (dict(tokens=None), -1, "null"), (dict(lp=None), -1, "null"), (dict(entropy=None), -1, "null"), (dict(top_tokens=None), -1, "null"),
    (dict(top_lp=None), -1, "null"),
])
def test_logprob_refusals(change, code, text):
    refused(logprobs(**change), code, text)


def test_host_memory_is_refused():
    """Well-formed calls whose pointers are not device memory."""
    for call in (quantize, norm, gated, linear, logprobs):
        refused(call(), -1, "not device memory")


def test_empty_calls_do_nothing():
    for call in (quantize, norm, gated, linear, logprobs):
        assert call(n=0) == 0


def test_workspace_sizes():
    b = ctypes.c_int64()
    assert lib().cq35_token_logprobs_workspace(1, 248320, 1, 20, ctypes.byref(b)) == 0 and b.value >= 0
    refused(lib().cq35_token_logprobs_workspace(1, 0, 1, 0, ctypes.byref(b)), -2, "logits")
    refused(lib().cq35_token_logprobs_workspace(1, 10, 1, 0, None), -1, "null")


def test_python_refusals():
    """The torch binding refuses tensors of another type, place or shape."""
    torch = pytest.importorskip("torch")
    import cq35
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    q = cq35.Int8Rows(torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        cq35.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        cq35.int8_linear(q, q)
    with pytest.raises(ValueError, match="GPU"):
        cq35.token_logprobs(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="bfloat16"):
        cq35.gated_quantize(x.half(), x)
    with pytest.raises(ValueError, match="dimensions"):
        cq35.norm_quantize(x[0], torch.ones(64))
    with pytest.raises(TypeError):
        cq35.quantize_rows(None)
    with pytest.raises(TypeError, match="pair"):
        cq35.int8_linear(None, q)
