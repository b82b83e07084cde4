"""The 4-bit products and the logit operators without a GPU: the library exports what the headers declare, its structs are the
binding's, bad arguments are refused on the host before any launch, the oracles agree with hand-computed values, and the quantiser
with its definition."""
import ctypes
import os
import re

import numpy as np
import pytest

import oracle
from conftest import REPO

torch = pytest.importorskip("torch")

from rwkv_next_amd import _lib  # noqa: E402
from rwkv_next_amd.kernels import int4_gemm as I4, sampler  # noqa: E402

FAKE = 0x100000  # a pointer that no refused call follows


def _declared(header, prefix):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", header)).read(), flags=re.S)
    return set(re.findall(r"^[A-Za-z_][\w \*]*?\b(%s_\w+)\s*\(" % prefix, text, flags=re.M))


def _fields(header, struct):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", header)).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % struct, text, flags=re.S).group(1)
    return [n.strip().lstrip("*") for decl in body.split(";") if decl.strip()
            for n in re.sub(r"^(const )?\w+ ", "", decl.strip()).split(",")]


@pytest.mark.parametrize("header,prefix,exported", [("w4a16.h", "w4a16", _lib.W4A16_EXPORTED),
                                                    ("logits.h", "logits", _lib.LOGITS_EXPORTED)])
def test_library_exports_what_the_headers_declare(header, prefix, exported):
    assert _declared(header, prefix) == set(exported)
    for n in exported:
        assert hasattr(_lib.load(), n), n


@pytest.mark.parametrize("header,struct,mirror", [
    ("w4a16.h", "w4a16_args", _lib.W4a16Args), ("logits.h", "logits_penalize_args", _lib.PenalizeArgs),
    ("logits.h", "logits_sample_args", _lib.SampleArgs)])
def test_structs_match(header, struct, mirror):
    assert _fields(header, struct) == [n for n, _ in mirror._fields_]
    assert getattr(_lib.load(), struct + "_size")() == ctypes.sizeof(mirror)


def test_constants_match():
    text = "".join(open(os.path.join(REPO, "include", h)).read() for h in ("w4a16.h", "logits.h"))
    for n in re.findall(r"#define ((?:W4A16|LOGITS)_\w+) ", text):
        value = re.search(r"#define %s (.*?)(?:/\*|$)" % n, text, flags=re.M).group(1).strip()
        if value:
            got = getattr(_lib, n, None)
            assert got is None or got == eval(value), n
    assert _lib.LOGITS_STATUS_ROW == 256 and _lib.LOGITS_STATUS_TOKEN == 512


def test_packed_arguments_are_the_struct():
    values = [i + 1 for i in range(len(_lib.SampleArgs._fields_))]
    assert _lib.pack_sample(*values) == bytes(_lib.SampleArgs(*values))
    values = [i + 1 for i in range(len(_lib.PenalizeArgs._fields_))]
    assert _lib.pack_penalize(*values) == bytes(_lib.PenalizeArgs(*values))
    values = [i + 1 for i in range(len(_lib.W4a16Args._fields_))]
    assert _lib.pack_w4a16(*values) == bytes(_lib.W4a16Args(*values))


def _set(a, kw):
    for n, v in kw.items():
        setattr(a, n, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    (dict(K=48), _lib.WKV7_ERR_SHAPE), (dict(K=0), _lib.WKV7_ERR_SHAPE), (dict(N=0), _lib.WKV7_ERR_SHAPE),
    (dict(M=-1), _lib.WKV7_ERR_SHAPE), (dict(group_k=16), _lib.WKV7_ERR_SHAPE), (dict(group_k=96), _lib.WKV7_ERR_SHAPE),
    (dict(group_k=0), _lib.WKV7_ERR_SHAPE), (dict(a_row_stride=248), _lib.WKV7_ERR_SHAPE),
    (dict(a_row_stride=(1 << 24) + 8), _lib.WKV7_ERR_SHAPE), (dict(out_row_stride=99), _lib.WKV7_ERR_SHAPE),
    (dict(a_row_stride=260), _lib.WKV7_ERR_ALIGN), (dict(a=FAKE + 8), _lib.WKV7_ERR_ALIGN),
    (dict(weight=FAKE + 4), _lib.WKV7_ERR_ALIGN), (dict(scales=FAKE + 2), _lib.WKV7_ERR_ALIGN),
    (dict(out=FAKE + 1), _lib.WKV7_ERR_ALIGN), (dict(out=FAKE + 2, out_dtype=_lib.W4A16_F32), _lib.WKV7_ERR_ALIGN),
    (dict(a=None), _lib.WKV7_ERR_NULL), (dict(weight=None), _lib.WKV7_ERR_NULL), (dict(out=None), _lib.WKV7_ERR_NULL),
    (dict(a_dtype=2), _lib.WKV7_ERR_ARG), (dict(out_dtype=3), _lib.WKV7_ERR_ARG), (dict(out_dtype=-1), _lib.WKV7_ERR_ARG),
    (dict(M=2 ** 31 - 1), _lib.WKV7_ERR_SHAPE), (dict(M=0, a=None, out=None), _lib.WKV7_OK),
])
def test_int4_refusals(kw, code):
    a = _lib.W4a16Args(FAKE, 256, FAKE, FAKE, FAKE, 100, 3, 100, 256, 128, 0, 0)
    assert _lib.load().w4a16_matmul(_set(a, kw), None) == code
    assert _lib.load().w4a16_matmul(None, None) == _lib.WKV7_ERR_NULL


def test_int4_helpers_refuse():
    lib, n, m = _lib.load(), ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert lib.w4a16_packed_size(128, 16, 48, ctypes.byref(n), ctypes.byref(m)) == _lib.WKV7_ERR_SHAPE
    assert lib.w4a16_packed_size(128, 16, 64, None, ctypes.byref(m)) == _lib.WKV7_ERR_NULL
    assert lib.w4a16_packed_size(160, 17, 32, ctypes.byref(n), ctypes.byref(m)) == 0
    assert (n.value, m.value) == (2 * 2 * 1024, 2 * 2 * 16 * 4 * 2)
    assert lib.w4a16_pack(None, FAKE, 128, 16, 64, FAKE, FAKE, None) == _lib.WKV7_ERR_NULL
    assert lib.w4a16_pack(FAKE, FAKE, 128, 16, 64, FAKE + 8, FAKE, None) == _lib.WKV7_ERR_ALIGN
    assert lib.w4a16_pack(FAKE, FAKE, 100, 16, 64, FAKE, FAKE, None) == _lib.WKV7_ERR_SHAPE
    assert lib.w4a16_dequantize(FAKE, FAKE, FAKE, 128, 16, 64, 3, None) == _lib.WKV7_ERR_ARG
    assert lib.w4a16_dequantize(FAKE, FAKE, FAKE + 2, 128, 16, 64, 2, None) == _lib.WKV7_ERR_ALIGN
    assert lib.w4a16_dequantize(FAKE, None, FAKE, 128, 16, 64, 2, None) == _lib.WKV7_ERR_NULL


def _penalize(**kw):
    a = _lib.PenalizeArgs(logits=FAKE, in_seq_stride=200, in_pos_stride=100, out=FAKE, out_seq_stride=200, out_pos_stride=100,
                          B=2, T=2, V=100, in_dtype=2, out_dtype=2)
    return _lib.load().logits_penalize(_set(a, kw), None)


@pytest.mark.parametrize("kw,code", [
    (dict(V=0), _lib.WKV7_ERR_SHAPE), (dict(B=-1), _lib.WKV7_ERR_SHAPE), (dict(n_bias=-1), _lib.WKV7_ERR_SHAPE),
    (dict(logits=None), _lib.WKV7_ERR_NULL), (dict(out=None), _lib.WKV7_ERR_NULL), (dict(n_bias=3), _lib.WKV7_ERR_NULL),
    (dict(in_dtype=3), _lib.WKV7_ERR_ARG), (dict(out_dtype=-1), _lib.WKV7_ERR_ARG),
    (dict(counts=FAKE, counts_stride=100, counts_rows=2, counts_dtype=2), _lib.WKV7_ERR_ARG),
    (dict(counts=FAKE, counts_stride=99, counts_rows=2), _lib.WKV7_ERR_SHAPE),
    (dict(counts=FAKE + 2, counts_stride=100, counts_rows=2), _lib.WKV7_ERR_ALIGN),
    (dict(drafts=FAKE, drafts_stride=0), _lib.WKV7_ERR_SHAPE),
    (dict(n_bias=3, bias_ids=FAKE, bias_values=FAKE, bias_stride=2), _lib.WKV7_ERR_SHAPE),
    (dict(mask=FAKE, mask_stride=3, mask_rows=4), _lib.WKV7_ERR_SHAPE),
    (dict(mask=FAKE + 1, mask_stride=4, mask_rows=4), _lib.WKV7_ERR_ALIGN),
    (dict(logits=FAKE + 2), _lib.WKV7_ERR_ALIGN), (dict(out=FAKE + 1, out_dtype=0), _lib.WKV7_ERR_ALIGN),
    (dict(V=2 ** 31 - 1, B=2 ** 20), _lib.WKV7_ERR_SHAPE), (dict(B=0, logits=None), _lib.WKV7_OK), (dict(T=0), _lib.WKV7_OK),
])
def test_penalize_refusals(kw, code):
    assert _penalize(**kw) == code
    assert _lib.load().logits_penalize(None, None) == _lib.WKV7_ERR_NULL


@pytest.mark.parametrize("kw,code", [
    (dict(V=0), _lib.WKV7_ERR_SHAPE), (dict(V=2 ** 21 + 1), _lib.WKV7_ERR_SHAPE), (dict(T=-1), _lib.WKV7_ERR_SHAPE),
    (dict(logits=None), _lib.WKV7_ERR_NULL), (dict(token=None), _lib.WKV7_ERR_NULL), (dict(dtype=4), _lib.WKV7_ERR_ARG),
    (dict(T=2, counts=FAKE, counts_stride=100, counts_rows=2), _lib.WKV7_ERR_ARG),
    (dict(counts=FAKE, counts_stride=10, counts_rows=2), _lib.WKV7_ERR_SHAPE),
    (dict(noise=FAKE + 1), _lib.WKV7_ERR_ALIGN), (dict(workspace=FAKE + 16), _lib.WKV7_ERR_ALIGN),
    (dict(workspace=None), _lib.WKV7_ERR_WORKSPACE), (dict(workspace_bytes=100), _lib.WKV7_ERR_WORKSPACE),
    (dict(B=0, token=None), _lib.WKV7_OK),
])
def test_sample_refusals(kw, code):
    a = _lib.SampleArgs(logits=FAKE, seq_stride=100, token=FAKE, workspace=FAKE, workspace_bytes=1 << 26, B=2, T=1, V=100, dtype=2)
    assert _lib.load().logits_sample(_set(a, kw), None) == code
    assert _lib.load().logits_sample(None, None) == _lib.WKV7_ERR_NULL


def test_sample_workspace_grows_with_the_rows_up_to_a_bound():
    n = ctypes.c_size_t(0)
    sizes = []
    for B in (0, 1, 64, 512, 5000):
        assert _lib.load().logits_sample_workspace_size(ctypes.byref(_lib.SampleArgs(B=B, T=1, V=100)), ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == _lib.LOGITS_SAMPLE_STATE_BYTES and sizes == sorted(sizes) and sizes[3] == sizes[4]


def test_python_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(2, 8)
    for f in (sampler.penalize_logits, sampler.sample_logits):
        with pytest.raises(ValueError, match="GPU"):
            f(x)
        with pytest.raises(TypeError):
            f(x.double())
    with pytest.raises(ValueError, match="GPU"):
        I4.prepack_int4(torch.zeros(32, 8, dtype=torch.uint8), torch.zeros(1, 8, dtype=torch.float16), 64)
    with pytest.raises(TypeError):
        I4.prepack_int4(torch.zeros(32, 8), torch.zeros(1, 8, dtype=torch.float16), 64)
    with pytest.raises(TypeError):
        I4.int4_matmul(x, I4.Int4Packed(x, x, 8, 8, 8))
    with pytest.raises(ValueError, match="GPU"):
        I4.int4_matmul(x.bfloat16(), I4.Int4Packed(x, x, 8, 8, 8))


# ----------------------------------------------------------------------------------------------------------------
# quantiser and oracles
# ----------------------------------------------------------------------------------------------------------------
def test_quantise():
    rng = np.random.default_rng(1)
    w = torch.from_numpy(rng.standard_normal((192, 37)).astype(np.float32))
    w[:, 5] = 0
    w[:64, 6] = -w[:64, 6].abs()
    for clip in (False, True):
        codes, scales, g = I4.quantize_int4(w, 64, clip_search=clip)
        assert codes.shape == (96, 37) and codes.dtype == torch.uint8 and scales.shape == (3, 37) and g == 64
        u = oracle.int4_ref.unpack_codes(codes.numpy()).astype(np.int64) - 8
        s = scales.numpy().astype(np.float32)[np.arange(192) // 64]
        want = np.clip(np.round(w.numpy() / s), -8, 7)
        assert np.array_equal(u, want)
        assert (u[:, 5] == 0).all() and np.isfinite(s).all() and (s > 0).all()
        err = np.square(oracle.int4_ref.dequantize_ref(codes.numpy(), scales.numpy(), 64) - w.numpy()).sum()
        if not clip:
            plain = err
            amax = np.abs(w.numpy()).reshape(3, 64, 37).max(1)
            assert np.array_equal(scales.numpy()[:, :5], (amax / 7.5).astype(np.float16)[:, :5])
    assert err < plain  # the clip search lowers the squared error
    assert I4.quantize_int4(w, 0)[2] == 192 and I4.quantize_int4(w, 1000)[2] == 192
    for bad in ((torch.zeros(48, 4), 32), (torch.zeros(64, 4), 48), (torch.zeros(2, 64, 4), 32)):
        with pytest.raises(ValueError):
            I4.quantize_int4(*bad)


def test_int4_oracle():
    u = np.arange(128).reshape(64, 2).astype(np.uint8) % 16
    codes = oracle.int4_ref.pack_codes(u)
    assert codes[0, 0] == (u[0, 0] | u[1, 0] << 4) and np.array_equal(oracle.int4_ref.unpack_codes(codes), u)
    scales = np.array([[0.5, 2.0], [1.0, -4.0]], np.float16)
    w = oracle.int4_ref.dequantize_ref(codes, scales, 32)
    assert w[0, 0] == 0.5 * (0 - 8) and w[1, 1] == 2.0 * (3 - 8) and w[40, 1] == -4.0 * (81 % 16 - 8)
    packed = oracle.int4_ref.packed_ref(codes)
    assert packed.shape == (1, 1, 64, 4)
    word = int(packed[0, 0, 17, 1])  # column 1, step 1: rows 32 + 8 ..
    assert [word >> (4 * j) & 15 for j in range(4)] == [int(u[40 + 2 * j, 1]) for j in range(4)]
    assert [word >> (16 + 4 * j) & 15 for j in range(4)] == [int(u[41 + 2 * j, 1]) for j in range(4)]
    assert int(packed[0, 0, 3, 0]) == 0x88888888 and int(packed[0, 0, 0, 2]) == 0x88888888  # past the weight
    s = oracle.int4_ref.packed_scales_ref(scales, 64, 32)
    assert s.shape == (1, 1, 16, 4) and s[0, 0, 1].tolist() == [2.0, -4.0, 0.0, 0.0]


def test_penalize_oracle():
    x = np.array([[[2.0, -2.0, 1.0, 0.5], [2.0, -2.0, 1.0, 0.5]]])
    y = oracle.logits_ref.penalize_ref(x, counts=np.array([[9, 9, 9, 9], [2, 1, 0, 0]]), slots=np.array([1]), repetition=2.0,
                                       presence=0.25, frequency=0.5, drafts=np.array([[2]]), bias_ids=np.array([[3, -1, 3]]),
                                       bias_values=np.array([[1.0, 5.0, 2.0]]),
                                       mask=np.array([[[0b1101], [0b1111]]], np.uint32))
    assert y[0, 0].tolist() == [2 / 2 - 1.25, -np.inf, 1.0, 3.5]
    assert y[0, 1].tolist() == [2 / 2 - 1.25, -2 * 2 - 0.75, 1 / 2 - 0.75, 3.5]


def test_choices_oracle():
    choices = lambda x, e, t=1.0, k=0, p=1.0, m=0.0: oracle.logits_ref.choices_ref(np.array(x), np.array(e), t, k, p, m, 1e-6)[0]  # noqa: E731
    x, ones = np.log([0.5, 0.3, 0.15, 0.05]), [1.0, 1.0, 1.0, 1.0]
    assert choices(x, ones) == {0} and choices(x, [1, 0.1, 1, 1]) == {1} and choices(x, [1, 1, 1, 0.001]) == {3}
    assert choices(x, [1, 1, 1, 0.001], k=3) == {0} and choices(x, [1, 1, 0.001, 1], k=3) == {2}
    assert choices(x, [1, 1, 0.001, 1e-9], p=0.9) == {2} and choices(x, [1, 1, 1e-9, 1e-9], p=0.79) == {0}
    assert choices(x, [1, 1e-3, 1e-9, 1], p=0.6) == {1} and choices(x, [1, 1e-9, 1, 1], p=0.4) == {0}
    assert choices(x, [1, 1, 1e-9, 1], m=0.31) == {0} and choices(x, [1, 1, 1e-9, 1], m=0.29) == {2}
    assert choices([0.0, 1.0, 1.0], [1.0, 1.0, 1.0]) == {1, 2}  # equal scores: either, the kernel's tests ask for the lower
    assert choices([0.0, 1.0, 1.0], [1.0, 1.0, 1e-9], k=1) == {1}  # equal logits: the lower is before the other
    assert choices(x, [1, 1e-9, 1, 1], t=0.0) == {0} and choices([-np.inf, np.nan], [1, 1]) == set()
    token, lp = oracle.logits_ref.choices_ref(x, None, 1.0, 0, 1.0, 0.0, 1e-6)
    assert token == {0} and np.allclose(np.exp(lp), [0.5, 0.3, 0.15, 0.05])
