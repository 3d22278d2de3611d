"""CPU: the host side of the language-model decode operators: 4-bit rounding of weights, argument
checks of the binding, status codes before envg_init."""
import numpy as np
import pytest

from invision_b200 import envg
from oracle import oracle as O
from tests import lm_ref as R


@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (5, 63, 64), (3, 300, 128), (7, 257, 32)])
def test_quantize_q4_within_half_a_step(N, K, group):
    rng = np.random.default_rng(K)
    w = (0.05 * rng.standard_normal((N, K)) + 0.02).astype(np.float32)
    w[0, : K // 3] = 0.0
    codes, scales, zeros = envg.quantize_q4(w, group)
    held = R.q4_weight(codes, scales, zeros, K, group)
    step = scales[:, np.arange(K) // group]
    # half a step, and half a step of the zero point's own rounding where a value would leave 0..15
    assert (np.abs(held - w) <= step * (1.0 + 1e-5)).all()
    assert np.abs(held - w).mean() <= 0.3 * step.mean()
    assert (held[w == 0] == 0).all() and zeros.max() <= 15
    bits = O.f32_to_bf16_rne(w)
    c2, s2, z2 = envg.quantize_q4(bits, group)
    c3, s3, z3 = envg.quantize_q4((bits.astype(np.uint32) << 16).view(np.float32), group)
    assert np.array_equal(c2, c3) and np.array_equal(s2, s3) and np.array_equal(z2, z3)


def test_quantize_q4_edges():
    codes, scales, zeros = envg.quantize_q4(np.zeros((2, 40), np.float32), 32)
    assert (R.q4_weight(codes, scales, zeros, 40, 32) == 0).all()
    w = np.array([[3e38, -3e38, 1.0]], np.float32)  # a span beyond fp32
    codes, scales, zeros = envg.quantize_q4(w, 32)
    assert np.isfinite(scales).all() and np.abs(R.q4_weight(codes, scales, zeros, 3, 32) - w).max() <= scales.max()
    for bad in (np.nan, np.inf):
        with pytest.raises(envg.EnvgError, match="not finite"):
            envg.quantize_q4(np.full((1, 3), bad, np.float32), 32)
    with pytest.raises(envg.EnvgError, match="group"):
        envg.quantize_q4(np.zeros((1, 3), np.float32), 16)
    with pytest.raises(TypeError):
        envg.quantize_q4(np.zeros((1, 3), np.float64))


def test_held_values_stay_near():
    """The cache's rounding as the tests state it: within half a step plus fp16 of the minimum."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 128)) * 3 + 1).astype(np.float32)
    y = R.kv_hold(x)
    g = x.reshape(50, 2, 64)
    step = (g.max(-1) - g.min(-1)) / 15
    assert (np.abs(y.reshape(g.shape) - g) <= step[..., None] * 0.51 + np.abs(g).max() * 2.0 ** -10).all()


def test_binding_refuses_before_any_call():
    f = np.zeros((2, 128), np.float32)
    with pytest.raises(ValueError, match="codes"):
        envg.Q4Weight(np.zeros((4, 10), np.uint8), np.zeros((4, 1), np.float32), K=64)
    with pytest.raises(ValueError, match="group"):
        envg.Q4Weight(np.zeros((4, 32), np.uint8), np.zeros((4, 1), np.float32), group=256)
    with pytest.raises(TypeError, match="scales"):
        envg.Q4Weight(np.zeros((4, 32), np.uint8), np.zeros((4, 1), np.float64), group=64)
    with pytest.raises(TypeError, match="adjacent"):
        envg._matrix(f[:, ::2], 2, 64, "x", envg.HOST_PTRS)
    with pytest.raises(TypeError, match="overlap"):
        envg._matrix(np.lib.stride_tricks.as_strided(f, (2, 64), (4, 4)), 2, 64, "x", envg.HOST_PTRS)
    assert envg._matrix(f[:, 3:60], 2, 57, "x", envg.HOST_PTRS)[1] == 128


def test_calls_before_init_return_state_error():
    try:
        import torch

        if torch.cuda.is_available():
            pytest.skip("checks the uninitialised state")
    except ImportError:
        pass
    L = envg.lib()
    for call in (L.envg_linear_q4, L.envg_qk_norm_rope, L.envg_kv4_append, L.envg_kv4_read, L.envg_attention_kv4):
        assert call(None, 0) == envg.ERR_STATE
    for go in (lambda: envg.KV4Cache(4, 16, 1, 128),
               lambda: envg.Q4Weight(np.zeros((4, 32), np.uint8), np.zeros((4, 1), np.float32), group=64)):
        with pytest.raises(envg.EnvgError) as e:
            go()
        assert e.value.code == envg.ERR_STATE
    assert L.envg_kv4_free(None) == envg.ERR_STATE and L.envg_q4weight_free(None) == envg.ERR_STATE
    assert L.envg_weight_upload_q4(None, None, None, 1, 1, 32, 0, 0, None) == envg.ERR_ARG


def test_packed_structures_match_the_header(tmp_path):
    """The binding packs each argument structure as the C compiler lays it out."""
    import os
    import subprocess

    names = {"envg_linear_q4_args": envg._LINEAR_Q4, "envg_qk_norm_rope_args": envg._QK_NORM_ROPE,
             "envg_kv4_rows": envg._KV4_ROWS, "envg_attention_kv4_args": envg._ATTENTION_KV4}
    last = {"envg_linear_q4_args": "epilogue", "envg_qk_norm_rope_args": "interleaved", "envg_kv4_rows": "q_len",
            "envg_attention_kv4_args": "scale"}
    src = tmp_path / "s.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"envgemm.h\"\nint main(void) {\n" + "".join(
        f'printf("%zu\\n", offsetof({n}, {last[n]}) + 4);\n' for n in names) + "return 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.dirname(envg.HEADER_PATH), str(src), "-o", str(tmp_path / "s")])
    sizes = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in sizes] == [st.size for st in names.values()]


def test_one_step_calls_leave_other_tensors_to_the_binding():
    """_views.call makes no call with a tensor that is not the CUDA matrix its spec asks for, nor with
    numbers that a field does not hold; it never throws through the interpreter."""
    import ctypes

    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError, match="CUDA"):
        envg._side(torch.zeros(1))
    if envg._views is None:
        pytest.skip("the torch extension was not built for this torch")
    calls = []
    fn = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int)(lambda p, f: calls.append(f) or 0)
    at, call = ctypes.cast(fn, ctypes.c_void_p).value, envg._views.call
    nested = torch.nested.as_nested_tensor([torch.zeros(2, 2), torch.zeros(3, 2)], layout=torch.strided)
    for t in (torch.zeros(2, 2), torch.empty(2, 2, device="meta"), nested, np.zeros((2, 2), np.float32), "x", None):
        assert call(at, 0, 0, "M", t, 2, 2) is None
        if t is not None:
            assert envg._views.matrix(t, 2, 2, 0) is None and envg._views.vector(t, 2, 0) is None
    for spec, operands, error in (("M", (), TypeError), ("q", (1, 2), TypeError), ("i", (1 << 40,), OverflowError),
                                  ("f", (1e300,), OverflowError), ("q", (1.5,), TypeError), ("p", (-1,), OverflowError)):
        with pytest.raises(error):
            call(at, 0, 0, spec, *operands)
    with pytest.raises(TypeError):
        call(at, 0, 0, "q" * 40, *range(40))  # more than a structure holds
    assert not calls


def _claim(torch, monkeypatch, t, device):
    """A tensor that says it lives on cuda:`device`; its memory is host memory, which nothing here reads."""
    import ctypes

    for name in ("init", "_lazy_init"):
        monkeypatch.setattr(torch.cuda, name, lambda: None)
    cap = torch.utils.dlpack.to_dlpack(t)
    get = ctypes.pythonapi.PyCapsule_GetPointer
    get.restype, get.argtypes = ctypes.c_void_p, [ctypes.py_object, ctypes.c_char_p]
    where = ctypes.cast(get(cap, b"dltensor") + 8, ctypes.POINTER(ctypes.c_int32))  # DLTensor: data, then device
    where[0], where[1] = 2, device  # kDLCUDA
    return torch._C._from_dlpack(cap)


def test_operands_of_several_devices_are_refused(monkeypatch):
    import ctypes

    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError, match="CUDA"):
        envg._side(torch.zeros(1))
    a, b, c = (_claim(torch, monkeypatch, torch.zeros(2, 4), d) for d in (0, 1, 0))
    n, m = _claim(torch, monkeypatch, torch.zeros(4), 1), _claim(torch, monkeypatch, torch.zeros(4), 0)
    monkeypatch.setattr(envg, "_device", 0)
    for views in (envg._views, None):  # the checks of the extension, and those in Python
        monkeypatch.setattr(envg, "_views", views)
        assert envg._matrix(a, 2, 4, "x", envg.DEVICE_PTRS) == (a.data_ptr(), 4)
        assert envg._vector(m, 4, "bias", envg.DEVICE_PTRS) == m.data_ptr()
        for look in (lambda: envg._matrix(b, 2, 4, "dst", envg.DEVICE_PTRS), lambda: envg._vector(n, 4, "dst", envg.DEVICE_PTRS),
                     lambda: envg._packed(b, 2, 4, "dst", envg.DEVICE_PTRS)):
            with pytest.raises(ValueError, match="dst: lives on cuda:1"):
                look()
    monkeypatch.undo()
    if envg._views is None:
        pytest.skip("the torch extension was not built for this torch")
    calls, refuse = [], 0
    fn = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int)(lambda p, f: calls.append(f) or 0)
    use = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p)(lambda d, s, p: calls.append((d, s, p)) or refuse)
    at, use_at = (ctypes.cast(f, ctypes.c_void_p).value for f in (fn, use))
    assert envg._views.call(at, use_at, 3, "MVM", a, 2, 4, m, 4, c, 2, 4) == 0
    assert calls == [(0, 0, None), 3]
    calls.clear()
    for operands in ((a, 2, 4, m, 4, b, 2, 4), (a, 2, 4, n, 4, c, 2, 4), (b, 2, 4, m, 4, c, 2, 4)):
        assert envg._views.call(at, use_at, 3, "MVM", *operands) is None
    assert not calls
    refuse = envg.ERR_ARG  # the library runs on another device
    assert envg._views.call(at, use_at, 3, "M", a, 2, 4) == envg.ERR_ARG
    assert calls == [(0, 0, None)]


@pytest.mark.parametrize("extra", [1, 2, 3])
def test_rows_at_odd_byte_distances_are_refused(extra):
    """Rows of a packed record: their distance in bytes is no multiple of an element, and a stride in
    elements would name other memory."""
    records = np.zeros(5, np.dtype([("x", np.float32, (8,)), ("tag", np.uint8, (extra,))]))
    assert records["x"].shape == (5, 8) and records["x"].strides == (32 + extra, 4)
    with pytest.raises(TypeError, match="x: rows .* bytes apart"):
        envg._matrix(records["x"], 5, 8, "x", envg.HOST_PTRS)
    with pytest.raises(TypeError):
        envg._packed(records["x"], 5, 8, "x", envg.HOST_PTRS)
    assert envg._matrix(records["x"][:1], 1, 8, "x", envg.HOST_PTRS)[1] == 8
    padded = np.zeros(5, np.dtype([("x", np.float32, (8,)), ("tag", np.uint8, (4,))]))
    assert envg._matrix(padded["x"], 5, 8, "x", envg.HOST_PTRS)[1] == 9


def test_read_only_outputs_are_refused():
    """An output that numpy holds to be read-only (a view of bytes, a file mapped for reading) is refused
    before any call; the same array is fine as an input."""
    import types

    ro, rw = np.frombuffer(bytes(4 * 2 * 64), np.float32).reshape(2, 64), np.zeros((2, 64), np.float32)
    n, table = np.array([2], np.int32), np.zeros((1, 1), np.int32)
    W = types.SimpleNamespace(N=64, K=64, layout=envg.LAYOUT_PLAIN, h=None)
    cache = object.__new__(envg.KV4Cache)
    cache.h, cache.kv_heads, cache.head_dim = None, 1, 64
    for call in (lambda: envg.linear_q4(ro, rw, W), lambda: envg.qk_norm_rope(ro, None, rw, None, None, None, None, None, 1, 0, 64),
                 lambda: envg.qk_norm_rope(None, ro, None, rw, None, None, None, None, 0, 1, 64),
                 lambda: cache.read(ro, rw, table, n, q_len=2), lambda: cache.read(rw, ro, table, n, q_len=2),
                 lambda: envg.attention_kv4(ro, rw, cache, table, n, 1, q_len=2)):
        with pytest.raises(ValueError, match="read-only"):
            call()
    for call in (lambda: envg.linear_q4(rw, ro, W), lambda: cache.append(ro, ro, table, n, q_len=2)):
        with pytest.raises(envg.EnvgError):  # as far as the library, which has no weight or cache here
            call()
