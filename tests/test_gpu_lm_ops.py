"""GPU: the language-model decode operators (4-bit linears, q/k norm + rotation, the paged 4-bit
cache, attention over it) against their formulas in 64 bits."""
import numpy as np
import pytest

from tests import lm_ref as R

pytestmark = pytest.mark.gpu

# Relative error of a whole output (2-norm): the operands' split and the fp32 sums leave a few 1e-7
# on random data; no rounding of x, of a score or of a weight to 16 bits fits below this.
REL = 3e-6


def _close(y, ref, tol, what=""):
    assert np.isfinite(y).all(), f"{what}: non-finite output"
    over = np.abs(y.astype(np.float64) - ref) - tol
    assert over.max() <= 0, f"{what}: {over.max():.3e} over the bound {tol.max():.3e}"
    assert R.rel(y, ref) <= REL, f"{what}: relative error {R.rel(y, ref):.3e}"


# ---- 4-bit linears ----------------------------------------------------------------------------

def _q4(N, K, group, zeros, seed):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)
    scales = (0.01 * (0.2 + rng.random((N, -(-K // group))))).astype(np.float32)
    z = rng.integers(0, 16, scales.shape, dtype=np.uint8) if zeros else None
    return codes, scales, z


Q4_CASES = [
    # M, K, N, group, zeros
    (1, 1, 1, 32, False), (1, 2, 17, 64, True), (1, 128, 16, 128, True), (1, 127, 15, 32, True),
    (2, 130, 33, 64, False), (3, 257, 50, 128, True), (4, 2560, 1024, 128, True), (5, 384, 48, 32, True),
    (7, 1000, 72, 64, False), (8, 4096, 40, 128, False), (9, 640, 100, 32, True), (12, 9728, 48, 32, True),
    (13, 2049, 31, 64, True), (16, 2560, 256, 64, True), (17, 320, 64, 128, False), (32, 1280, 96, 64, True),
    (33, 513, 40, 32, True), (64, 640, 200, 64, True), (64, 16384, 32, 128, True), (1, 16384, 2000, 128, True),
    (4, 11000, 64, 32, False), (100, 300, 70, 64, True), (1, 64, 5000, 32, False),
]


@pytest.mark.parametrize("M,K,N,group,zeros", Q4_CASES)
def test_linear_q4_vs_formula(gpu, M, K, N, group, zeros):
    codes, scales, z = _q4(N, K, group, zeros, M * 31 + K + N)
    rng = np.random.default_rng(M + K + N)
    x = rng.standard_normal((M, K)).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32) if N % 2 else None
    W = gpu.Q4Weight(codes, scales, z, K=K, group=group)
    y = np.full((M, N), np.nan, np.float32)
    gpu.linear_q4(y, x, W, bias=b)
    ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), b, groups=-(-K // group))
    _close(y, ref, tol, f"{M}x{K}x{N}")


@pytest.mark.parametrize("M,K,half,group", [(1, 2560, 608, 128), (2, 100, 1, 32), (5, 513, 37, 64), (16, 640, 136, 32), (40, 256, 20, 128)])
def test_linear_q4_silu_gate(gpu, M, K, half, group):
    codes, scales, z = _q4(2 * half, K, group, True, M)
    rng = np.random.default_rng(M + K)
    x = rng.standard_normal((M, K)).astype(np.float32)
    b = rng.standard_normal(2 * half).astype(np.float32) if half % 2 else None
    W = gpu.Q4Weight(codes, scales, z, K=K, group=group, layout=gpu.LAYOUT_GATE_UP)
    y = np.full((M, half), np.nan, np.float32)
    gpu.linear_q4(y, x, W, bias=b)
    ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), b, gate_up=True, groups=-(-K // group))
    over = np.abs(y - ref) - tol
    assert np.isfinite(y).all() and over.max() <= 0, over.max()
    assert R.rel(y, ref) <= 2 * REL


@pytest.mark.parametrize("M", [1, 6, 20])
def test_linear_q4_gated_residual_strides_and_canaries(gpu, M):
    import torch

    K, N, group = 384, 150, 64
    codes, scales, z = _q4(N, K, group, True, 5)
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, K)).astype(np.float32)
    h = rng.standard_normal((M, N)).astype(np.float32)
    b, g = rng.standard_normal((2, N)).astype(np.float32)
    cu = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    W = gpu.Q4Weight(cu(codes), cu(scales), cu(z), K=K, group=group)
    # views with odd strides and offsets: rows that are not 16-byte aligned
    xb = torch.full((M, K + 9), float("nan"), device="cuda")
    yb = torch.full((M, N + 7), 7.0, device="cuda")
    xb[:, 3 : 3 + K], yb[:, 5 : 5 + N] = cu(x), cu(h)
    gpu.linear_q4(yb[:, 5 : 5 + N], xb[:, 3 : 3 + K], W, bias=cu(b), epilogue=gpu.EPI_GATED_RESIDUAL, gate=cu(g))
    got = yb.cpu().numpy()
    y, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), b, groups=K // group)
    ref = h + g * y
    over = np.abs(got[:, 5 : 5 + N] - ref) - (np.abs(g) * tol + 2.0 ** -23 * (np.abs(ref) + np.abs(g * y)))
    assert over.max() <= 0, over.max()
    assert (got[:, :5] == 7.0).all() and (got[:, 5 + N :] == 7.0).all()


@pytest.mark.parametrize("M", [3, 10])
def test_linear_q4_value_ranges(gpu, M):
    """Rows of very different sizes, a wide range inside one row, a zero row, one with a NaN."""
    K, N, group = 640, 64, 64
    codes, scales, z = _q4(N, K, group, True, 11)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0] *= 1e30
    x[1] *= np.exp(rng.uniform(-40, 0, K)).astype(np.float32)
    x[2] = 0.0
    if M > 3:
        x[3] *= 1e-30
        x[4, 17] = np.nan
        x[5, 600] = np.inf
    W = gpu.Q4Weight(codes, scales, z, K=K, group=group)
    y = np.zeros((M, N), np.float32)
    gpu.linear_q4(y, x, W)
    fine = [i for i in range(M) if np.isfinite(x[i]).all()]
    ref, tol = R.linear(x[fine], R.q4_weight(codes, scales, z, K, group), groups=K // group)
    for i, r in enumerate(fine):
        _close(y[r], ref[i], tol[i], f"row {r}")
    for r in set(range(M)) - set(fine):
        assert not np.isfinite(y[r]).any(), r


def test_linear_q4_host_equals_device_and_repeats(gpu):
    import torch

    M, K, N, group = 4, 2560, 1000, 128
    codes, scales, z = _q4(N, K, group, True, 2)
    x = np.random.default_rng(1).standard_normal((M, K)).astype(np.float32)
    W = gpu.Q4Weight(codes, scales, z, K=K, group=group)
    y = np.zeros((M, N), np.float32)
    gpu.linear_q4(y, x, W)
    xd, s = torch.from_numpy(x).cuda(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):  # a stream of the caller's, repeated
        for _ in range(3):
            yd = torch.full((M, N), float("nan"), device="cuda")
            gpu.linear_q4(yd, xd, W, sync=False)
            s.synchronize()
            assert np.array_equal(yd.cpu().numpy(), y)
    # a captured graph replays the call
    g, yg = torch.cuda.CUDAGraph(), torch.zeros((M, N), device="cuda")
    with torch.cuda.graph(g):
        gpu.linear_q4(yg, xd, W, sync=False)
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(yg.cpu().numpy(), y)


def test_quantize_q4_round_trip(gpu):
    """quantize_q4 -> upload -> linear: within half a step of every weight of the float linear."""
    rng = np.random.default_rng(8)
    K, N, group = 300, 40, 64
    w = (0.02 * rng.standard_normal((N, K))).astype(np.float32)
    codes, scales, z = gpu.quantize_q4(w, group)
    held = R.q4_weight(codes, scales, z, K, group)
    x = rng.standard_normal((2, K)).astype(np.float32)
    y = np.zeros((2, N), np.float32)
    gpu.linear_q4(y, x, gpu.Q4Weight(codes, scales, z, K=K, group=group))
    ref, tol = R.linear(x, held, groups=-(-K // group))
    _close(y, ref, tol)


def test_linear_q4_refusals(gpu):
    codes, scales, z = _q4(64, 128, 64, True, 0)
    W = gpu.Q4Weight(codes, scales, z, K=128, group=64)
    x, y = np.zeros((2, 128), np.float32), np.zeros((2, 64), np.float32)
    L = gpu.lib()
    call = lambda **k: L.envg_linear_q4(gpu._LINEAR_Q4.pack(*{**dict(dst=y.ctypes.data, ldd=64, x=x.ctypes.data, ldx=128, W=W.h.value, bias=0, gate=0, M=2, K=128, N=64, epi=0), **k}.values()), 0)  # noqa: E731
    assert call() == gpu.OK
    for bad in (dict(K=127), dict(N=63), dict(M=-1), dict(ldx=127), dict(ldd=63), dict(epi=gpu.EPI_BIAS), dict(epi=gpu.EPI_SILU_GATE),
                dict(epi=gpu.EPI_GATED_RESIDUAL), dict(epi=9), dict(dst=0), dict(x=0), dict(x=y.ctypes.data, ldx=128)):
        assert call(**bad) == gpu.ERR_ARG, bad
        assert gpu.last_error()
    assert L.envg_linear_q4(None, 0) == gpu.ERR_ARG
    assert call(W=0) == gpu.ERR_STATE
    assert call(M=0, dst=0, x=0) == gpu.OK
    plain = gpu.Weight(np.zeros((64, 128), np.uint16))
    assert call(W=plain.h.value) == gpu.ERR_STATE  # a 16-bit weight is not a 4-bit one, and the other way
    assert L.envg_linear(y.ctypes.data, x.ctypes.data, W.h, None, 2, 128, 64, 0, None, 0) == gpu.ERR_STATE
    with pytest.raises(ValueError, match="group"):
        gpu.Q4Weight(codes, scales, z, K=128, group=48)
    with pytest.raises(gpu.EnvgError, match="even number"):
        gpu.Q4Weight(codes[:63], scales[:63], z[:63], K=128, group=64, layout=gpu.LAYOUT_GATE_UP)
    with pytest.raises(gpu.EnvgError, match="above 15"):
        gpu.Q4Weight(codes, scales, np.full_like(z, 16), K=128, group=64)
    with pytest.raises(TypeError):
        gpu.linear_q4(y, x.astype(np.float64), W)
    with pytest.raises(ValueError):
        gpu.linear_q4(y[:1], x, W)
    W.free()
    with pytest.raises(gpu.EnvgError):
        gpu.linear_q4(y, x, W)


# ---- norm + rotation ---------------------------------------------------------------------------

@pytest.mark.parametrize("T,H,KVH,hd", [(1, 32, 8, 128), (5, 3, 1, 64), (16, 4, 4, 256), (7, 2, 0, 96), (3, 0, 5, 8), (130, 6, 2, 24), (33, 1, 1, 200), (300, 24, 24, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope_vs_formula(gpu, T, H, KVH, hd, interleaved):
    rng = np.random.default_rng(T + hd)
    q, k = rng.standard_normal((T, H * hd)).astype(np.float32), (3 * rng.standard_normal((T, KVH * hd))).astype(np.float32)
    wq = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    wk = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if T % 2 else None
    ang = np.arange(400)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    pos = rng.integers(0, 400, T).astype(np.int32) if T != 16 else None
    at = pos if pos is not None else 9 + np.arange(T)
    qo, ko = (np.full_like(q, np.nan) if H else None), (np.full_like(k, np.nan) if KVH else None)
    gpu.qk_norm_rope(qo, ko, q if H else None, k if KVH else None, wq, wk, cos, sin, H, KVH, hd, positions=pos, pos0=9,
                     interleaved=interleaved)
    for got, x, n, w in ((qo, q, H, wq), (ko, k, KVH, wk)):
        if n:
            ref, tol = R.norm_rope(x, n, hd, w, cos, sin, at, interleaved, 1e-6)
            _close(got, ref, tol)


def test_qk_norm_rope_in_place_strided_and_norm_only(gpu):
    """q and k as slices of one fused projection's rows, rotated in place; odd offsets; no tables."""
    import torch

    T, H, KVH, hd = 9, 4, 2, 64
    rng = np.random.default_rng(0)
    for off in (0, 3):
        buf = torch.from_numpy(rng.standard_normal((T, off + (H + 2 * KVH) * hd + 5)).astype(np.float32)).cuda()
        before = buf.cpu().numpy()
        q, k = buf[:, off : off + H * hd], buf[:, off + H * hd : off + (H + KVH) * hd]
        ang = np.arange(64)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
        cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        gpu.qk_norm_rope(q, k, q, k, None, None, torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), H, KVH, hd, pos0=2)
        got = buf.cpu().numpy()
        a, b = off + H * hd, off + (H + KVH) * hd
        for lo, hi, n in ((off, a, H), (a, b, KVH)):
            ref, tol = R.norm_rope(before[:, lo:hi], n, hd, None, cos, sin, 2 + np.arange(T), False, 1e-6)
            _close(got[:, lo:hi], ref, tol)
        assert np.array_equal(got[:, :off], before[:, :off]) and np.array_equal(got[:, b:], before[:, b:])
    x = rng.standard_normal((T, H * hd)).astype(np.float32)
    y = np.zeros_like(x)
    gpu.qk_norm_rope(y, None, x, None, None, None, None, None, H, 0, hd, eps=0.5)
    ref, tol = R.norm_rope(x, H, hd, None, None, None, None, False, 0.5)
    _close(y, ref, tol)
    z = np.zeros((2, hd), np.float32)  # a head of zeros stays zeros
    gpu.qk_norm_rope(z, None, z.copy(), None, None, None, None, None, 1, 0, hd)
    assert (z == 0).all()


def test_qk_norm_rope_refusals(gpu):
    import torch

    x = np.zeros((2, 128), np.float32)
    t = np.zeros((4, 64), np.float32)
    go = lambda **k: gpu.qk_norm_rope(**{**dict(q_dst=x, k_dst=None, q=x, k=None, q_weight=None, k_weight=None, cos=t, sin=t, heads=1, kv_heads=0, head_dim=128), **k})  # noqa: E731
    go()
    for bad, code in ((dict(pos0=3), gpu.ERR_ARG), (dict(pos0=-1), gpu.ERR_ARG), (dict(eps=-1.0), gpu.ERR_ARG),
                      (dict(positions=np.array([0, 4], np.int32)), gpu.ERR_ARG), (dict(positions=np.array([0, -1], np.int32)), gpu.ERR_ARG),
                      (dict(sin=None), gpu.ERR_ARG), (dict(head_dim=12, cos=None, sin=None), gpu.ERR_UNSUPPORTED),
                      (dict(head_dim=264, heads=0, cos=None, sin=None), gpu.ERR_UNSUPPORTED)):
        with pytest.raises(gpu.EnvgError) as e:
            go(**bad)
        assert e.value.code == code, bad
    with pytest.raises(ValueError):
        go(heads=2)
    with pytest.raises(TypeError):
        go(positions=np.zeros(2, np.int64))
    # on the device a position out of range is clamped and reported by the next synchronising call
    xd, td = torch.ones((2, 128), device="cuda"), torch.ones((4, 64), device="cuda")
    with pytest.raises(gpu.EnvgError, match="position") as e:
        gpu.qk_norm_rope(xd, None, xd, None, None, None, td, td, 1, 0, 128, positions=torch.tensor([1, 4], dtype=torch.int32, device="cuda"))
    assert e.value.code == gpu.ERR_ARG
    gpu.sync()


# ---- the cache ----------------------------------------------------------------------------------

def _tables(rng, lens, page, spare=2):
    per = max(1, max(-(-max(n, 1) // page) for n in lens))
    ids = rng.permutation(len(lens) * per + spare).astype(np.int32)
    table = np.full((len(lens), per), -7, np.int32)  # entries past a sequence's end name nothing
    at = 0
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = ids[at : at + m]
        at += m
    return table, len(ids)


@pytest.mark.parametrize("lens,q_len,page,KVH,hd", [([1], 1, 16, 1, 64), ([5, 40, 17], 1, 16, 2, 128), ([100, 33], 33, 48, 3, 64), ([3, 0, 20], 8, 32, 2, 128), ([700], 600, 128, 8, 128)])
def test_kv4_append_read_bit_for_bit(gpu, lens, q_len, page, KVH, hd):
    rng = np.random.default_rng(sum(lens) + hd)
    table, pages = _tables(rng, lens, page)
    n = len(lens) * q_len
    k = (rng.standard_normal((n, KVH * hd)) * np.exp(rng.uniform(-5, 5, (n, 1)))).astype(np.float32)
    v = (5 + rng.standard_normal((n, KVH * hd))).astype(np.float32)
    k[0, :64] = 1.25  # a group without a span
    v[-1, -64:] = -3e5 * rng.random(64)  # beyond fp16
    c = gpu.KV4Cache(pages, page, KVH, hd)
    cl = np.asarray(lens, np.int32)
    c.append(k, v, table, cl, q_len=q_len)
    ko, vo = np.full_like(k, np.nan), np.full_like(v, np.nan)
    c.read(ko, vo, table, cl, q_len=q_len)
    there = (np.repeat(cl, q_len) - q_len + np.tile(np.arange(q_len), len(lens)) >= 0)[:, None]
    for got, x in ((ko, k), (vo, v)):
        ref = R.kv_hold(x.reshape(n, KVH, hd)).reshape(n, -1) * there
        assert np.array_equal(got, ref.astype(np.float32))


@pytest.mark.parametrize("lens,q_len,page,KVH,hd", [([1500, 1190], 1201, 48, 8, 128), ([2401], 2401, 16, 16, 64), ([12003], 12001, 64, 8, 128), ([6001, 5999], 6001, 32, 16, 64)])
def test_kv4_append_read_long_runs(gpu, lens, q_len, page, KVH, hd):
    """Enough tokens that a thread takes two or four of them: odd lengths, runs that begin inside a tile
    and before the first token."""
    test_kv4_append_read_bit_for_bit(gpu, lens, q_len, page, KVH, hd)


def test_kv4_append_keeps_its_neighbours_and_holds_nan(gpu):
    """Token by token equals all at once; a NaN stays in its group; device strides."""
    import torch

    rng = np.random.default_rng(5)
    L, page, KVH, hd = 50, 16, 2, 64
    table, pages = _tables(rng, [L], page)
    x = rng.standard_normal((L, 2 * KVH * hd + 3)).astype(np.float32)
    x[20, 3] = np.nan
    x[21, KVH * hd + 2] = np.inf
    xd, td = torch.from_numpy(x).cuda(), torch.from_numpy(table).cuda()
    k, v = xd[:, 1 : 1 + KVH * hd], xd[:, 1 + KVH * hd : 1 + 2 * KVH * hd]
    a, b = gpu.KV4Cache(pages, page, KVH, hd), gpu.KV4Cache(pages, page, KVH, hd)
    ln = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")  # noqa: E731
    a.append(k, v, td, ln(L), q_len=L)
    for i in range(L):
        b.append(k[i : i + 1], v[i : i + 1], td, ln(i + 1), sync=False)
    out = [[torch.empty((L, KVH * hd), device="cuda") for _ in range(2)] for _ in range(2)]
    a.read(*out[0], td, ln(L), q_len=L)
    b.read(*out[1], td, ln(L), q_len=L)
    for i, y in enumerate((k, v)):
        got = out[0][i].cpu().numpy()
        assert np.array_equal(got, out[1][i].cpu().numpy(), equal_nan=True)
        assert np.array_equal(got, R.kv_hold(y.cpu().numpy().reshape(L, KVH, hd)).reshape(L, -1), equal_nan=True)
    assert np.isnan(out[0][0].cpu().numpy()[20]).sum() == 64


def test_kv4_refusals(gpu):
    import torch

    for args, code in (((4, 15, 1, 128), gpu.ERR_ARG), ((4, 0, 1, 128), gpu.ERR_ARG), ((0, 16, 1, 128), gpu.ERR_ARG),
                       ((4, 16, 0, 128), gpu.ERR_ARG), ((4, 16, 1, 96), gpu.ERR_UNSUPPORTED)):
        with pytest.raises(gpu.EnvgError) as e:
            gpu.KV4Cache(*args)
        assert e.value.code == code, args
    c = gpu.KV4Cache(4, 16, 2, 64)
    k = np.zeros((1, 128), np.float32)
    t, n = np.array([[0, 1]], np.int32), np.array([17], np.int32)
    q, o = np.zeros((1, 256), np.float32), np.zeros((1, 256), np.float32)
    c.append(k, k, t, n)
    gone = np.array([[-1, 1]], np.int32)  # the append touches its own page alone
    c.append(k, k, gone, n)
    with pytest.raises(gpu.EnvgError):
        gpu.attention_kv4(o, q, c, gone, n, 4)
    for table, lens in ((t, np.array([33], np.int32)), (t, np.array([-1], np.int32)), (np.array([[0, 4]], np.int32), n)):
        for go in (lambda: c.append(k, k, table, lens), lambda: gpu.attention_kv4(o, q, c, table, lens, 4)):
            with pytest.raises(gpu.EnvgError) as e:
                go()
            assert e.value.code == gpu.ERR_ARG
    for bad in (dict(heads=3), dict(window=-1), dict(sinks=-1), dict(max_ctx=-1), dict(scale=0.0)):
        with pytest.raises((gpu.EnvgError, ValueError)):
            gpu.attention_kv4(o, q, c, t, n, **{**dict(heads=4), **bad})
    with pytest.raises(gpu.EnvgError):
        gpu.attention_kv4(q, q, c, t, n, 4)
    with pytest.raises(TypeError):
        c.append(k, k, t.astype(np.int64), n)
    # the device reports what only it can see, reads nothing out of bounds and works on
    cu = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    for table, lens, word in ((np.array([[0, 99]], np.int32), n, "page"), (t, np.array([40], np.int32), "length")):
        with pytest.raises(gpu.EnvgError, match=word):
            gpu.attention_kv4(cu(o), cu(q), c, cu(table), cu(lens), 4)
        with pytest.raises(gpu.EnvgError, match=word):
            c.append(cu(k), cu(k), cu(table), cu(lens))
    gpu.attention_kv4(o, q, c, t, n, 4)
    c.free()
    with pytest.raises(gpu.EnvgError):
        c.append(k, k, t, n)


# ---- attention over the cache ---------------------------------------------------------------------

def _held(gpu, rng, lens, page, KVH, hd, scale_v=None, bad=None):
    """A filled cache and the values it holds: (cache, table, [k per sequence], [v ...])."""
    full = max(max(lens), 1)
    table, pages = _tables(rng, [max(n, 1) for n in lens], page)
    c = gpu.KV4Cache(pages, page, KVH, hd)
    ks, vs = [], []
    for b, n in enumerate(lens):
        m = (table[b] >= 0).sum() * page  # the whole of its pages, past its length too
        k = rng.standard_normal((m, KVH, hd)).astype(np.float32) * (0.5 + 1.5 * rng.random((KVH, hd)).astype(np.float32))
        v = rng.standard_normal((m, KVH, hd)).astype(np.float32)
        if scale_v is not None:
            v *= scale_v(m)[:, None, None].astype(np.float32)
        k[n:], v[n:] = np.nan, np.inf  # what lies behind a sequence's end is never looked at
        if bad is not None:
            k[bad(b, m)], v[bad(b, m)] = np.nan, np.nan
        c.append(k.reshape(m, -1), v.reshape(m, -1), table[b : b + 1], np.array([m], np.int32), q_len=m)
        ks.append(R.kv_hold(k)), vs.append(R.kv_hold(v))
    assert full <= table.shape[1] * page
    return c, table, ks, vs


def _check_attention(gpu, rng, c, table, ks, vs, lens, q_len, H, hd, window=0, sinks=0, qscale=1.0, max_ctx=0, scale=None):
    B = len(lens)
    q = (qscale * rng.standard_normal((B * q_len, H * hd))).astype(np.float32)
    out = np.full_like(q, np.nan)
    gpu.attention_kv4(out, q, c, table, np.asarray(lens, np.int32), H, q_len=q_len, max_ctx=max_ctx, window=window, sinks=sinks, scale=scale)
    for b, n in enumerate(lens):
        rows = slice(b * q_len, (b + 1) * q_len)
        pos = n - q_len + np.arange(q_len)
        ref, tol = R.attention(q[rows].reshape(q_len, H, hd), ks[b][:n], vs[b][:n], pos, window, sinks, scale or hd ** -0.5)
        got = out[rows].reshape(q_len, H, hd)
        assert (got[pos < 0] == 0).all()
        assert np.isfinite(got).all()
        over = np.abs(got - ref) - tol
        assert over.max() <= 0, (b, over.max())
        if n:
            # scores of size |x| carry their own rounding into the weights
            assert R.rel(got, ref) <= 4 * REL * max(1.0, qscale), (b, R.rel(got, ref))
    return out


ATTN = [
    # lens, q_len, page, H, KVH, hd, window, sinks
    ([1], 1, 16, 1, 1, 64, 0, 0),
    ([1, 2, 15, 16, 17, 31, 33], 1, 16, 4, 1, 128, 0, 0),
    ([0, 5, 0], 1, 16, 2, 2, 64, 0, 0),
    ([300, 64, 129], 1, 48, 8, 2, 128, 0, 0),
    ([1000], 1, 64, 32, 8, 128, 0, 0),
    ([2000, 777], 1, 128, 6, 2, 64, 0, 0),      # three heads to a kv head
    ([513], 1, 32, 16, 1, 128, 0, 0),           # sixteen heads to a kv head
    ([100, 40], 2, 16, 5, 1, 128, 0, 0),
    ([100, 3, 0], 5, 16, 4, 2, 64, 0, 0),       # more new tokens than a sequence has
    ([70, 200], 64, 32, 4, 2, 128, 0, 0),
    ([33], 33, 16, 3, 3, 64, 0, 0),
    ([500, 20, 90], 1, 16, 4, 2, 128, 64, 4),
    ([500], 1, 16, 4, 2, 128, 1, 0),
    ([500], 1, 16, 4, 2, 64, 17, 1),
    ([500], 1, 64, 4, 2, 128, 100, 33),
    ([500], 1, 64, 4, 2, 128, 100, 450),        # sinks up to and into the window
    ([500, 90], 40, 16, 4, 2, 128, 30, 5),      # a chunk longer than the window
    ([300], 20, 32, 4, 4, 64, 16, 20),
    ([3000], 1, 16, 2, 1, 128, 2047, 3),
]


@pytest.mark.parametrize("lens,q_len,page,H,KVH,hd,window,sinks", ATTN)
def test_attention_kv4_vs_formula(gpu, lens, q_len, page, H, KVH, hd, window, sinks):
    rng = np.random.default_rng(sum(lens) + H + hd + window)
    c, table, ks, vs = _held(gpu, rng, lens, page, KVH, hd)
    _check_attention(gpu, rng, c, table, ks, vs, lens, q_len, H, hd, window, sinks, max_ctx=max(lens))


def test_attention_kv4_value_ranges(gpu):
    """Sharp and flat scores, values whose sizes differ by tokens and sequences, a given scale."""
    rng = np.random.default_rng(1)
    lens = [400, 90]
    for qscale in (0.0, 1e-4, 30.0):
        c, table, ks, vs = _held(gpu, rng, lens, 32, 2, 128)
        _check_attention(gpu, rng, c, table, ks, vs, lens, 1, 8, 128, qscale=qscale)
    for sv in (lambda m: np.exp(rng.uniform(-7, 7, m)), lambda m: np.full(m, 1e-3), lambda m: np.where(np.arange(m) < 5, 1e4, 1.0), lambda m: np.zeros(m)):
        c, table, ks, vs = _held(gpu, rng, lens, 16, 2, 64, scale_v=sv)
        _check_attention(gpu, rng, c, table, ks, vs, lens, 1, 4, 64, scale=0.3)
    # rows of queries with very different sizes do not touch one another
    c, table, ks, vs = _held(gpu, rng, [200], 16, 1, 64)
    q = rng.standard_normal((1, 4 * 64)).astype(np.float32)
    q[0, :64] *= 1e-20
    q[0, 64:128] = np.nan
    out = np.zeros_like(q)
    gpu.attention_kv4(out, q, c, table, np.array([200], np.int32), 4)
    ref, tol = R.attention(q.reshape(1, 4, 64)[:, [0, 2, 3]], ks[0][:200], vs[0][:200], [199], 0, 0, 64 ** -0.5)
    assert (np.abs(out.reshape(1, 4, 64)[:, [0, 2, 3]] - ref) <= tol).all()
    assert np.isnan(out.reshape(4, 64)[1]).all()


def test_attention_kv4_hidden_tokens_may_hold_anything(gpu):
    """NaN in tokens that the window hides, and pages the table no longer names."""
    rng = np.random.default_rng(2)
    lens, page = [400, 333], 16
    hide = lambda b, m: np.arange(6, lens[b] - 50)  # noqa: E731
    c, table, ks, vs = _held(gpu, rng, lens, page, 2, 128, bad=hide)
    _check_attention(gpu, rng, c, table, ks, vs, lens, 1, 4, 128, window=50, sinks=6)
    _check_attention(gpu, rng, c, table, ks, vs, lens, 3, 4, 128, window=40, sinks=2)
    for b, n in enumerate(lens):
        table[b, 1 : (n - 50) // page] = -1
    _check_attention(gpu, rng, c, table, ks, vs, lens, 1, 4, 128, window=50, sinks=6)
    # a NaN that is seen is not hidden either
    c2, t2, _, _ = _held(gpu, rng, [40], page, 1, 64, bad=lambda b, m: [3])
    out = np.zeros((1, 64), np.float32)
    gpu.attention_kv4(out, rng.standard_normal((1, 64)).astype(np.float32), c2, t2, np.array([40], np.int32), 1)
    assert np.isnan(out).all()


def test_attention_kv4_beyond_4_gib_strides_streams_repeats(gpu):
    import torch

    rng = np.random.default_rng(3)
    KVH, hd, page, H = 8, 128, 1024, 16
    pages = 4200  # 1.18 MB each: the last ones lie past 4 GiB
    c = gpu.KV4Cache(pages, page, KVH, hd)
    table = np.array([[4199, 3], [0, 4198]], np.int32)
    lens = np.array([1500, 1100], np.int32)
    L = 2048
    k, v = (rng.standard_normal((2 * L, KVH * hd)).astype(np.float32) for _ in range(2))
    c.append(k, v, table, np.full(2, L, np.int32), q_len=L)
    q = rng.standard_normal((2, H * hd + 11)).astype(np.float32)
    qd = torch.from_numpy(q).cuda()[:, 3 : 3 + H * hd]
    od = torch.full((2, H * hd + 6), 9.0, device="cuda")
    td, ld = torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    with torch.cuda.stream(s):
        for _ in range(3):
            gpu.attention_kv4(od[:, 1 : 1 + H * hd], qd, c, td, ld, H, max_ctx=1500, sync=False)
            s.synchronize()
            got.append(od.cpu().numpy())
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    assert (got[0][:, 0] == 9).all() and (got[0][:, 1 + H * hd :] == 9).all()
    for b in range(2):
        kk, vv = (R.kv_hold(x.reshape(2, L, KVH, hd)[b, : lens[b]]) for x in (k, v))
        ref, tol = R.attention(q[b, 3 : 3 + H * hd].reshape(1, H, hd), kk, vv, [lens[b] - 1], 0, 0, hd ** -0.5)
        y = got[0][b, 1 : 1 + H * hd].reshape(1, H, hd)
        assert (np.abs(y - ref) <= tol).all() and R.rel(y, ref) <= 4 * REL


# ---- all of them together ------------------------------------------------------------------------

def test_decode_example_matches_plain_layers(gpu):
    """examples/decode_q4.py at a small size: each layer within fp32 rounding of its plain form.  A key
    whose rounding falls the other way in the two forms cannot occur: both read the cache's values."""
    import importlib.util
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("decode_q4", os.path.join(root, "examples", "decode_q4.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    worst, _ = ex.run(layers=2, batch=3, steps=3, hidden=256, heads=6, kv_heads=2, head_dim=64, mlp=384, page=16, prompt=20)
    assert worst <= 2e-5, worst


def test_random_shapes_against_formulas(gpu):
    """A sweep of drawn sizes over all four operators, odd ones among them."""
    rng = np.random.default_rng(77)
    for _ in range(12):
        group = int(rng.choice([32, 64, 128]))
        M, K, half = int(rng.integers(1, 70)), int(rng.integers(1, 3000)), int(rng.integers(1, 300))
        codes, scales, z = _q4(2 * half, K, group, bool(rng.integers(2)), int(rng.integers(1 << 30)))
        x = rng.standard_normal((M, K)).astype(np.float32)
        gu = bool(rng.integers(2))
        W = gpu.Q4Weight(codes, scales, z, K=K, group=group, layout=gpu.LAYOUT_GATE_UP if gu else gpu.LAYOUT_PLAIN)
        y = np.full((M, half if gu else 2 * half), np.nan, np.float32)
        gpu.linear_q4(y, x, W)
        ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), gate_up=gu, groups=-(-K // group))
        assert np.isfinite(y).all() and (np.abs(y - ref) - tol).max() <= 0 and R.rel(y, ref) <= 2 * REL, (M, K, half, group, gu)
    for _ in range(12):
        hd, KVH, per = int(rng.choice([64, 128])), int(rng.integers(1, 5)), int(rng.integers(1, 10))
        B, q_len, page = int(rng.integers(1, 5)), int(rng.integers(1, 12)), int(rng.choice([16, 48, 80]))
        lens = [int(v) for v in rng.integers(0, 400, B)]
        window = int(rng.choice([0, 1, 20, 130]))
        c, table, ks, vs = _held(gpu, rng, lens, page, KVH, hd)
        _check_attention(gpu, rng, c, table, ks, vs, lens, q_len, KVH * per, hd, window, int(rng.integers(0, 40)) if window else 0)


def test_torch_operands_are_the_same_by_every_way_of_the_binding(gpu, monkeypatch):
    """One-step calls, checks of each operand by the extension, checks in Python: equal bits, equal
    refusals; strided operands, a side stream, a subclass of torch.Tensor."""
    import torch

    from invision_b200 import envg

    rng = np.random.default_rng(77)
    H, KVH, hd, B, L = 4, 2, 64, 3, 70
    table, pages = _tables(rng, [L] * B, 16)
    w = gpu.Q4Weight(*gpu.quantize_q4(rng.standard_normal((H * hd, 96)).astype(np.float32), 32), K=96, group=32)
    cud = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    x, bias = cud(rng.standard_normal((B, 96)).astype(np.float32)), cud(rng.standard_normal(H * hd).astype(np.float32))
    kv = cud(rng.standard_normal((B, 2 * KVH * hd + 5)).astype(np.float32))
    nw, ang = cud(rng.standard_normal(hd).astype(np.float32)), cud(rng.standard_normal((L, hd // 2)).astype(np.float32))
    td, pos = cud(table), cud(np.array([0, 7, 69], np.int32))
    stream = torch.cuda.Stream()

    def layer():
        cache = gpu.KV4Cache(pages, 16, KVH, hd)
        lens = cud(np.array([1, 1, 1], np.int32))
        q, k = torch.empty(B, H * hd + 3, device="cuda"), torch.empty(B, KVH * hd, device="cuda")
        ko, vo, out = torch.empty_like(k), torch.empty_like(k), torch.empty(B, H * hd, device="cuda")
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            gpu.linear_q4(q[:, : H * hd], x, w, bias=torch.nn.Parameter(bias), sync=False)
            gpu.qk_norm_rope(q[:, : H * hd], k, q[:, : H * hd], kv[:, : KVH * hd], nw, nw, ang.cos(), ang.sin(), H, KVH, hd, positions=pos, sync=False)
            cache.append(k, kv[:, KVH * hd : 2 * KVH * hd], td, lens, sync=False)
            cache.read(ko, vo, td, lens, sync=False)
            gpu.attention_kv4(out, q[:, : H * hd], cache, td, lens, H, window=5, sinks=1, sync=True)
        with pytest.raises(ValueError, match="x"):
            gpu.linear_q4(out, x[:, :95], w)
        with pytest.raises(TypeError):
            gpu.linear_q4(out, x.double(), w)
        with pytest.raises(ValueError, match="ctx_lens|q|dst"):
            gpu.attention_kv4(out[:2], q[:, : H * hd], cache, td, lens, H)
        with pytest.raises(TypeError):
            cache.append(k.cpu(), k, td, lens)
        return [t.cpu().numpy() for t in (q[:, : H * hd], k, ko, vo, out)]

    ways = [layer()]
    assert envg._Tensor is torch.Tensor  # the extension is there
    monkeypatch.setattr(envg, "_Tensor", None)
    ways.append(layer())
    monkeypatch.setattr(envg, "_views", None)
    ways.append(layer())
    for other in ways[1:]:
        for a, b in zip(ways[0], other):
            assert np.isfinite(a).all() and np.array_equal(a, b)


def test_kv4_length_beyond_the_table_leaves_its_sequence_alone(gpu):
    """A length that only the device can see to be out of range: nothing is appended for its sequence and
    what the cache holds stays; reads and attention give zeros there; the other sequences are served."""
    import torch

    rng = np.random.default_rng(4)
    KVH, hd, page, H, B = 2, 64, 16, 4, 3
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(B, 2)
    c = gpu.KV4Cache(6, page, KVH, hd)
    dev = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    full, some = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([32, 32, 32], [32, 30, 32]))

    def held():
        k, v = (torch.empty(B * 32, KVH * hd, device="cuda") for _ in range(2))
        c.read(k, v, table, full, q_len=32)
        return k.cpu().numpy().reshape(B, 32, -1), v.cpu().numpy().reshape(B, 32, -1)

    c.append(dev(B * 32, KVH * hd), dev(B * 32, KVH * hd), table, full, q_len=32)
    before = held()
    q, out, good = dev(B * 3, H * hd), torch.full((B * 3, H * hd), 7.0, device="cuda"), torch.empty(B * 3, H * hd, device="cuda")
    k, v = dev(B * 3, KVH * hd), dev(B * 3, KVH * hd)
    for n in (33, 2 ** 31 - 1, -1):
        lens = torch.tensor([32, n, 32], dtype=torch.int32, device="cuda")
        gpu.attention_kv4(good, q, c, table, some, H, q_len=3)
        with pytest.raises(gpu.EnvgError, match="length"):
            gpu.attention_kv4(out, q, c, table, lens, H, q_len=3)
        o, g = out.cpu().numpy().reshape(B, 3, -1), good.cpu().numpy().reshape(B, 3, -1)
        assert (o[1] == 0).all() and np.array_equal(o[[0, 2]], g[[0, 2]])
        ko, vo = (torch.full((B * 3, KVH * hd), 7.0, device="cuda") for _ in range(2))
        with pytest.raises(gpu.EnvgError, match="length"):
            c.read(ko, vo, table, lens, q_len=3)
        for got, was in zip((ko, vo), before):
            got = got.cpu().numpy().reshape(B, 3, -1)
            assert (got[1] == 0).all() and np.array_equal(got[[0, 2]], was[[0, 2], 29:])
        with pytest.raises(gpu.EnvgError, match="length"):
            c.append(k, v, table, lens, q_len=3)
        after = held()
        for got, was, x in zip(after, before, (k, v)):
            assert np.array_equal(got[1], was[1]) and np.array_equal(got[[0, 2], :29], was[[0, 2], :29])
            new = R.kv_hold(x.cpu().numpy().reshape(B, 3, KVH, hd)).reshape(B, 3, -1)
            assert np.array_equal(got[[0, 2], 29:], new[[0, 2]])
        before = after


def test_qk_norm_rope_in_place_with_another_stride_is_refused(gpu):
    """On the device the rows of one would be overwritten while they are read; one row, or one stride, is fine."""
    import torch

    buf = torch.randn(1024, device="cuda")
    wide, narrow = buf.view(4, 256), buf[:512].view(4, 128)
    before = buf.clone()
    for q, k in (((narrow, wide[:, :128]), (None, None)), ((None, None), (wide[:, :128], narrow))):
        n = [1 if t[0] is not None else 0 for t in (q, k)]
        with pytest.raises(gpu.EnvgError, match="in place") as e:
            gpu.qk_norm_rope(q[0], k[0], q[1], k[1], None, None, None, None, *n, 128)
        assert e.value.code == gpu.ERR_ARG
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    gpu.qk_norm_rope(narrow[:1], None, wide[:1, :128], None, None, None, None, None, 1, 0, 128)
    gpu.qk_norm_rope(wide[:, 128:], None, wide[:, 128:], None, None, None, None, None, 1, 0, 128)
    for rows in (buf[:128].view(1, 128), wide[:, 128:]):
        assert torch.allclose((rows * rows).mean(-1), torch.ones(len(rows), device="cuda"), atol=1e-5)
    x = np.random.default_rng(0).standard_normal(1024).astype(np.float32)  # host pointers: copied, any strides
    w, n = x.reshape(4, 256), x[:512].reshape(4, 128)
    ref, tol = R.norm_rope(w[:, :128].copy(), 1, 128, None, None, None, None, False, 1e-6)
    gpu.qk_norm_rope(n, None, w[:, :128], None, None, None, None, None, 1, 0, 128)
    _close(n, ref, tol)
