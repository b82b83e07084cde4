"""The products with an epilogue, the gated delta rule and the slot operators without a GPU: the library exports what the headers
declare, its structs are the binding's, bad arguments are refused on the host before any launch, and the oracle agrees with
hand-computed values."""
import ctypes
import os
import re

import numpy as np
import pytest

import oracle
from conftest import REPO

torch = pytest.importorskip("torch")

from rwkv_next_amd import _lib  # noqa: E402

FAKE = 0x100000  # a pointer that no refused call follows


def _text(header):
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", header)).read(), flags=re.S)


@pytest.mark.parametrize("header,prefix,exported", [
    ("dense.h", "dense", _lib.DENSE_EXPORTED), ("delta.h", "delta", _lib.DELTA_EXPORTED), ("slots.h", "slots", _lib.SLOTS_EXPORTED)])
def test_library_exports_what_the_headers_declare(header, prefix, exported):
    declared = set(re.findall(r"^[A-Za-z_][\w \*]*?\b(%s_\w+)\s*\(" % prefix, _text(header), flags=re.M))
    assert declared == set(exported)
    for n in exported:
        assert hasattr(_lib.load(), n), n


@pytest.mark.parametrize("header,struct,mirror", [
    ("dense.h", "dense_args", _lib.DenseArgs), ("delta.h", "delta_args", _lib.DeltaArgs), ("slots.h", "slots_cache", _lib.SlotsCache)])
def test_structs_match(header, struct, mirror):
    body = re.search(r"typedef struct %s \{(.*?)\}" % struct, _text(header), flags=re.S).group(1)
    fields = [n.strip().lstrip("*") for decl in body.split(";") if decl.strip()
              for n in re.sub(r"^(const )?\w+ ", "", decl.strip()).split(",")]
    assert fields == [n.rstrip("_") for n, _ in mirror._fields_]
    assert getattr(_lib.load(), struct + "_size")() == ctypes.sizeof(mirror)


def test_constants_match():
    for h in ("dense.h", "delta.h", "slots.h"):
        for n, value in re.findall(r"#define ((?:DENSE|DELTA|SLOTS)_\w+) (.+)", _text(h)):
            assert getattr(_lib, n) == eval(value), n
    bits = [v for n, v in vars(_lib).items() if "_STATUS_" in n and not n.endswith("MAX_SEQS")]
    assert len(set(bits)) == len(bits) and all(b & (b - 1) == 0 for b in bits)


def test_packed_arguments_are_the_struct():
    for pack, mirror in ((_lib.pack_dense, _lib.DenseArgs), (_lib.pack_delta, _lib.DeltaArgs)):
        values = [i + 1 for i in range(len(mirror._fields_))]
        assert pack(*values) == bytes(mirror(*values))


def _set(a, kw):
    for n, v in kw.items():
        setattr(a, n, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    (dict(K=48), _lib.WKV7_ERR_SHAPE), (dict(K=0), _lib.WKV7_ERR_SHAPE), (dict(N=0), _lib.WKV7_ERR_SHAPE),
    (dict(M=-1), _lib.WKV7_ERR_SHAPE), (dict(a_row_stride=248), _lib.WKV7_ERR_SHAPE),
    (dict(a_row_stride=(1 << 24) + 8), _lib.WKV7_ERR_SHAPE), (dict(out_row_stride=99), _lib.WKV7_ERR_SHAPE),
    (dict(residual=FAKE, residual_row_stride=99), _lib.WKV7_ERR_SHAPE),
    (dict(a_row_stride=260), _lib.WKV7_ERR_ALIGN), (dict(a=FAKE + 8), _lib.WKV7_ERR_ALIGN), (dict(weight=FAKE + 8), _lib.WKV7_ERR_ALIGN),
    (dict(out=FAKE + 1), _lib.WKV7_ERR_ALIGN), (dict(out=FAKE + 2, out_dtype=2), _lib.WKV7_ERR_ALIGN),
    (dict(bias=FAKE + 1, bias_dtype=0), _lib.WKV7_ERR_ALIGN), (dict(residual=FAKE + 2, residual_dtype=2, residual_row_stride=100), _lib.WKV7_ERR_ALIGN),
    (dict(a=None), _lib.WKV7_ERR_NULL), (dict(weight=None), _lib.WKV7_ERR_NULL), (dict(out=None), _lib.WKV7_ERR_NULL),
    (dict(dtype=2), _lib.WKV7_ERR_ARG), (dict(out_dtype=3), _lib.WKV7_ERR_ARG), (dict(activation=7), _lib.WKV7_ERR_ARG),
    (dict(activation=-1), _lib.WKV7_ERR_ARG), (dict(bias=FAKE, bias_dtype=3), _lib.WKV7_ERR_ARG),
    (dict(residual=FAKE, residual_dtype=-1), _lib.WKV7_ERR_ARG), (dict(M=0), _lib.WKV7_OK)])
def test_dense_refuses(kw, code):
    a = _lib.DenseArgs(a=FAKE, a_row_stride=256, weight=FAKE, out=FAKE, out_row_stride=100, M=4, N=100, K=256)
    assert _lib.load().dense_matmul(_set(a, kw), None) == code
    assert _lib.load().dense_matmul(None, None) == _lib.WKV7_ERR_NULL


def test_dense_sizes():
    n = ctypes.c_size_t(0)
    lib = _lib.load()
    assert lib.dense_packed_size(96, 17, ctypes.byref(n)) == 0 and n.value == 3 * 2 * 1024
    assert lib.dense_packed_size(1 << 20, 1 << 20, ctypes.byref(n)) == 0 and n.value == 1 << 41
    for K, N in ((33, 16), (0, 16), (32, 0), (-32, 16)):
        assert lib.dense_packed_size(K, N, ctypes.byref(n)) == _lib.WKV7_ERR_SHAPE
        assert lib.dense_pack(FAKE, 1, 1, K, N, FAKE, None) == _lib.WKV7_ERR_SHAPE
    assert lib.dense_packed_size(32, 16, None) == _lib.WKV7_ERR_NULL
    assert lib.dense_pack(None, 1, 1, 32, 16, FAKE, None) == _lib.WKV7_ERR_NULL
    assert lib.dense_pack(FAKE, 1, 1, 32, 16, FAKE + 8, None) == _lib.WKV7_ERR_ALIGN


@pytest.mark.parametrize("kw,code", [
    (dict(K=32), _lib.WKV7_ERR_SHAPE), (dict(K=256), _lib.WKV7_ERR_SHAPE), (dict(V=24), _lib.WKV7_ERR_SHAPE),
    (dict(V=0), _lib.WKV7_ERR_SHAPE), (dict(V=272), _lib.WKV7_ERR_SHAPE), (dict(Hv=3), _lib.WKV7_ERR_SHAPE),
    (dict(Hk=0), _lib.WKV7_ERR_SHAPE), (dict(Hk=8), _lib.WKV7_ERR_SHAPE), (dict(num_seqs=-1), _lib.WKV7_ERR_SHAPE), (dict(T=-1), _lib.WKV7_ERR_SHAPE),
    (dict(total_tokens=19), _lib.WKV7_ERR_SHAPE), (dict(total_tokens=(1 << 30) + 1), _lib.WKV7_ERR_SHAPE),
    (dict(num_seqs=1 << 30, T=0), _lib.WKV7_ERR_SHAPE),
    (dict(q_stride=120), _lib.WKV7_ERR_SHAPE), (dict(v_stride=248), _lib.WKV7_ERR_SHAPE), (dict(g_stride=3), _lib.WKV7_ERR_SHAPE),
    (dict(beta_stride=3), _lib.WKV7_ERR_SHAPE), (dict(o_stride=248), _lib.WKV7_ERR_SHAPE), (dict(k_stride=(1 << 24) + 8), _lib.WKV7_ERR_SHAPE),
    (dict(h0_rows=-1), _lib.WKV7_ERR_SHAPE), (dict(q_stride=132), _lib.WKV7_ERR_ALIGN), (dict(o_stride=260), _lib.WKV7_ERR_ALIGN),
    (dict(q=FAKE + 8), _lib.WKV7_ERR_ALIGN), (dict(o=FAKE + 8), _lib.WKV7_ERR_ALIGN), (dict(g=FAKE + 2), _lib.WKV7_ERR_ALIGN),
    (dict(h0=FAKE + 8), _lib.WKV7_ERR_ALIGN), (dict(ht=FAKE + 4), _lib.WKV7_ERR_ALIGN), (dict(snapshots=FAKE + 4), _lib.WKV7_ERR_ALIGN),
    (dict(q=None), _lib.WKV7_ERR_NULL), (dict(beta=None), _lib.WKV7_ERR_NULL),
    (dict(h0=None, h0_idx=FAKE), _lib.WKV7_ERR_ARG), (dict(ht=None, ht_idx=FAKE), _lib.WKV7_ERR_ARG), (dict(token_len=-2), _lib.WKV7_ERR_ARG),
    (dict(snapshots=FAKE, cu_seqlens=FAKE, T=0), _lib.WKV7_ERR_ARG), (dict(num_seqs=0), _lib.WKV7_OK)])
def test_delta_refuses(kw, code):
    a = _lib.DeltaArgs(q=FAKE, k=FAKE, v=FAKE, q_stride=128, k_stride=128, v_stride=256, g=FAKE, beta=FAKE, g_stride=4, beta_stride=4,
                       o=FAKE, o_stride=256, h0=FAKE, h0_rows=4, ht=FAKE, ht_rows=4, total_tokens=20, num_seqs=4, T=5, Hk=2, Hv=4,
                       K=64, V=64, scale=1.0, token_len=-1)
    assert _lib.load().delta_run(_set(a, kw), None) == code
    assert _lib.load().delta_run(None, None) == _lib.WKV7_ERR_NULL
    assert _lib.load().delta_workspace_size(ctypes.byref(a), None) == _lib.WKV7_ERR_NULL


def _cache(**kw):
    c = dict(from_=FAKE, to=FAKE, from_layer_stride=4096, from_slot_stride=64, to_layer_stride=4096, to_slot_stride=64, row_bytes=64, layers=2)
    return _lib.SlotsCache(**dict(c, **kw))


@pytest.mark.parametrize("kw,code", [
    (dict(from_=None), _lib.WKV7_ERR_NULL), (dict(to=None), _lib.WKV7_ERR_NULL), (dict(row_bytes=-1), _lib.WKV7_ERR_SHAPE),
    (dict(layers=-1), _lib.WKV7_ERR_SHAPE), (dict(from_slot_stride=63), _lib.WKV7_ERR_SHAPE), (dict(to_slot_stride=63), _lib.WKV7_ERR_SHAPE),
    (dict(to_layer_stride=-64), _lib.WKV7_ERR_SHAPE), (dict(layers=1 << 30), _lib.WKV7_ERR_SHAPE), (dict(layers=0, to=None), _lib.WKV7_OK),
    (dict(row_bytes=0), _lib.WKV7_OK)])
def test_slots_refuse_a_cache(kw, code):
    c = (_lib.SlotsCache * 1)(_cache(**kw))
    assert _lib.load().slots_copy(c, 1, FAKE, FAKE, 3, 8, 8, None, None) == code


def test_slots_refuse():
    lib, c = _lib.load(), (_lib.SlotsCache * 17)(*[_cache()] * 17)
    E = _lib
    assert lib.slots_copy(c, 17, FAKE, FAKE, 3, 8, 8, None, None) == E.WKV7_ERR_SHAPE
    assert lib.slots_copy(c, 1, FAKE, FAKE, 1025, 8, 8, None, None) == E.WKV7_ERR_SHAPE
    assert lib.slots_copy(c, 1, FAKE, FAKE, -1, 8, 8, None, None) == E.WKV7_ERR_SHAPE
    assert lib.slots_copy(c, 1, FAKE, FAKE, 1, 1 << 31, 8, None, None) == E.WKV7_ERR_SHAPE
    assert lib.slots_copy(c, 1, FAKE, None, 1, 8, 8, None, None) == E.WKV7_ERR_NULL
    assert lib.slots_copy(None, 1, FAKE, FAKE, 1, 8, 8, None, None) == E.WKV7_ERR_NULL
    assert lib.slots_copy(c, 1, None, None, 0, 8, 8, None, None) == E.WKV7_OK
    assert lib.slots_copy(c, 0, FAKE, FAKE, 3, 8, 8, None, None) == E.WKV7_OK
    assert lib.slots_free(c, 1, None, 2, 8, None, None) == E.WKV7_ERR_NULL
    assert lib.slots_free(c, 1, FAKE, 65536, 8, None, None) == E.WKV7_ERR_SHAPE
    assert lib.slots_free(c, 1, None, 0, 8, None, None) == E.WKV7_OK
    assert lib.slots_compact(c, 1, None, 8, None, None, None) == E.WKV7_ERR_NULL
    assert lib.slots_compact(c, 1, FAKE, 8193, None, None, None) == E.WKV7_ERR_SHAPE


def test_entry_points_refuse_host_tensors():
    from rwkv_next_amd import kernels
    w = torch.zeros(64, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        kernels.prepack_dense(w)
    with pytest.raises(ValueError):
        kernels.dense_matmul(torch.zeros(2, 64, dtype=torch.bfloat16), kernels.DensePacked(w.reshape(-1), 64, 16))
    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        kernels.gated_delta(q, q, q, torch.zeros(1, 2, 1), torch.zeros(1, 2, 1))
    with pytest.raises(ValueError):
        kernels.SlotCaches(torch.zeros(2, 3, 4))


def test_oracle_by_hand():
    ref = oracle.delta_ref
    q = k = np.array([[[1.0, 0.0]], [[0.6, 0.8]]])
    v = np.array([[[2.0]], [[3.0]]])
    o, states = ref.gated_delta_ref(q, k, v, np.log([[0.5], [0.25]]), np.array([[1.0], [0.5]]), np.array([[[4.0], [8.0]]]), scale=1.0)
    # after one token: (4, 8) / 2 -> k reads 2, writes 2 - 2 = 0: (2, 4).  After two: (0.5, 1) -> reads 0.3 + 0.8, writes 0.95 k
    assert np.allclose(states[1], [[[2.0], [4.0]]]) and np.allclose(states[2], [[[0.5 + 0.57], [1.0 + 0.76]]])
    assert np.allclose(o, [[[2.0]], [[0.6 * 1.07 + 0.8 * 1.76]]])
    y, x = ref.dense_ref([[1.0, -2.0]], [[1.0, 0.0], [0.0, 1.0]], [0.5, 0.5], "relu2", [[1.0, 1.0]])
    assert np.allclose(x, [[1.5, -1.5]]) and np.allclose(y, [[3.25, 1.0]])
    assert abs(ref.ACTIVATIONS["gelu"](np.array(1.0)) - 0.8413447460685429) < 1e-15
