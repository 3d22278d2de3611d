"""GPU: what the language-model decode operators keep of their operands' bits: groups of channels
of very different sizes, rows near the ends of fp32's range, NaN that has to come through."""
import numpy as np
import pytest

from tests import lm_ref as R

pytestmark = pytest.mark.gpu

# 2-norm of a group's error over the group's own norm, for scores up to 16 in log2 units.  A score is
# rounded to fp32 about four times at that size (2^-20 / sqrt(12) each, 5.5e-7 together, times ln 2 in
# the weight), a weight by its exponential (2^-22), its product with V's scale to 22 bits of the
# group's largest and by up to some tens of fp32 additions (2e-7): together below 1e-6.
REL_GROUP = 2e-6


def _fill(gpu, rng, lens, page, k, v):
    """A cache holding k and v ([sequences][tokens, KVH, hd]) in shuffled pages: (cache, table)."""
    KVH, hd = k[0].shape[1:]
    per = -(-max(lens) // page)
    table = rng.permutation(len(lens) * per).astype(np.int32).reshape(len(lens), per)
    c = gpu.KV4Cache(len(lens) * per, page, KVH, hd)
    for b, n in enumerate(lens):
        c.append(k[b].reshape(n, -1), v[b].reshape(n, -1), table[b : b + 1], np.array([n], np.int32), q_len=n)
    return c, table


@pytest.mark.parametrize("ratio", [1.0, 1e-1, 1e2, 1e3, 1e-4, 1e6])
@pytest.mark.parametrize("lens,q_len,H,KVH,window,sinks", [([700, 333], 1, 8, 2, 0, 0), ([700, 333], 1, 16, 2, 0, 0),
                                                           ([400], 5, 4, 2, 100, 7), ([33], 3, 2, 2, 0, 0)])
def test_attention_kv4_value_groups_of_different_size(gpu, lens, q_len, H, KVH, window, sinks, ratio):
    """Channels 0..63 and 64..127 of V differ in size by `ratio`: each keeps its own precision."""
    hd = 128
    rng = np.random.default_rng(H + q_len)
    size = np.repeat([ratio ** 0.5, ratio ** -0.5], 64).astype(np.float32)
    k = [rng.standard_normal((n, KVH, hd)).astype(np.float32) for n in lens]
    v = [rng.standard_normal((n, KVH, hd)).astype(np.float32) * size for n in lens]
    c, table = _fill(gpu, rng, lens, 16, k, v)
    q = rng.standard_normal((len(lens) * q_len, H * hd)).astype(np.float32)
    out = np.full_like(q, np.nan)
    gpu.attention_kv4(out, q, c, table, np.asarray(lens, np.int32), H, q_len=q_len, window=window, sinks=sinks)
    for b, n in enumerate(lens):
        rows = slice(b * q_len, (b + 1) * q_len)
        ref = R.attention_exact(q[rows].reshape(q_len, H, hd), R.kv_hold(k[b]), R.kv_hold(v[b]), n - q_len + np.arange(q_len),
                                window, sinks, hd ** -0.5)
        got = out[rows].reshape(q_len, H, hd)
        for g in (np.s_[..., :64], np.s_[..., 64:]):
            assert R.rel(got[g], ref[g]) <= REL_GROUP, (b, ratio, R.rel(got[g], ref[g]))


@pytest.mark.parametrize("n,q_len,H,KVH,window", [(2000, 1, 4, 1, 0), (2000, 1, 8, 1, 0), (90, 1, 1, 1, 0), (300, 2, 4, 1, 250), (1600, 3, 4, 2, 1500)])
@pytest.mark.parametrize("what", ["key", "value", "infinite score"])
def test_attention_kv4_seen_nan_comes_through_beside_large_scores(gpu, n, q_len, H, KVH, window, what):
    """A token with a NaN whose weight underflows beside one of a far larger score, whichever warps and
    CTAs the two fall to: the row (a NaN key) or the channels of its group (a NaN value) are NaN."""
    hd = 128
    first = max(0, n - q_len + 1 - window) + q_len if window else 0
    for at, big in ((first, n - q_len - 1), (n - q_len - 3, first + 2), (first + 7, first + 41), ((first + n) // 2, first + 1)):
        rng = np.random.default_rng(at)
        q = rng.standard_normal((q_len, H * hd)).astype(np.float32)
        k = rng.standard_normal((n, KVH, hd)).astype(np.float32)
        v = rng.standard_normal((n, KVH, hd)).astype(np.float32)
        for h in range(H):  # every row scores this token by some hundreds above the others
            k[big, h // (H // KVH)] += 40.0 * np.sign(q[:, h * hd : (h + 1) * hd]).sum(0)
        q *= 6.0
        if what == "key":
            k[at] = np.nan
        elif what == "value":
            v[at, :, 70] = np.nan
        else:
            q[:] = np.abs(q) * 1e36
            k[at] = 3e4
        c, table = _fill(gpu, rng, [n], 16, [k], [v])
        out = np.zeros_like(q)
        gpu.attention_kv4(out, q, c, table, np.array([n], np.int32), H, q_len=q_len, window=window)
        out = out.reshape(q_len, H, hd)
        if what == "value":
            assert np.isfinite(out[..., :64]).all() and np.isnan(out[..., 64:]).all(), (at, big)
        else:
            assert np.isnan(out).all(), (at, big)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 6, 12])
@pytest.mark.parametrize("size", [1e-25, 1e-30, 1e-33, 1e-36, 3e-38, 1e-40, 1e-43])
def test_linear_q4_keeps_tiny_rows(gpu, M, size):
    """Rows whose largest value is near fp32's smallest normal number, or below it, against large
    scales: x is what fp32 holds, and no bit of it is lost.  One row of ordinary size beside them."""
    K, N, group = 640, 48, 64
    rng = np.random.default_rng(M)
    codes = rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    z = rng.integers(0, 16, (N, K // group), dtype=np.uint8)
    scales = (1e27 * (0.2 + rng.random((N, K // group)))).astype(np.float32)
    x = (size * rng.standard_normal((M, K))).astype(np.float32)
    if M > 1:
        x[M // 2] = rng.standard_normal(K).astype(np.float32)
    y = np.zeros((M, N), np.float32)
    gpu.linear_q4(y, x, gpu.Q4Weight(codes, scales, z, K=K, group=group))
    ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), groups=K // group)
    assert np.isfinite(y).all()
    for r in range(M):
        assert (np.abs(y[r] - ref[r]) <= tol[r]).all() and R.rel(y[r], ref[r]) <= 3e-6, (r, R.rel(y[r], ref[r]))


@pytest.mark.parametrize("ratio", [1e2, 1e-3, 1e4, 1e-5, 1e6])
@pytest.mark.parametrize("lens,q_len,H,KVH,window,sinks", [([700, 333], 1, 8, 2, 0, 0), ([700, 333], 1, 16, 2, 0, 0),
                                                           ([400], 5, 4, 2, 100, 7)])
def test_attention_kv4_query_groups_of_different_size(gpu, lens, q_len, H, KVH, window, sinks, ratio):
    """Channels 0..63 and 64..127 of q differ in size by `ratio`, those of K the other way, so that both
    count alike in a score: each keeps its own precision."""
    hd = 128
    rng = np.random.default_rng(H + q_len)
    size = np.repeat([ratio ** 0.5, ratio ** -0.5], 64).astype(np.float32)
    k = [rng.standard_normal((n, KVH, hd)).astype(np.float32) / size for n in lens]
    v = [rng.standard_normal((n, KVH, hd)).astype(np.float32) for n in lens]
    c, table = _fill(gpu, rng, lens, 16, k, v)
    q = (rng.standard_normal((len(lens) * q_len, H, hd)).astype(np.float32) * size).reshape(-1, H * hd)
    out = np.full_like(q, np.nan)
    gpu.attention_kv4(out, q, c, table, np.asarray(lens, np.int32), H, q_len=q_len, window=window, sinks=sinks)
    for b, n in enumerate(lens):
        rows = slice(b * q_len, (b + 1) * q_len)
        ref = R.attention_exact(q[rows].reshape(q_len, H, hd), R.kv_hold(k[b]), R.kv_hold(v[b]), n - q_len + np.arange(q_len),
                                window, sinks, hd ** -0.5)
        got = out[rows].reshape(q_len, H, hd)
        assert R.rel(got, ref) <= REL_GROUP, (b, ratio, R.rel(got, ref))


@pytest.mark.parametrize("M", [1, 2, 3, 4, 6, 12])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6, 1e8])
def test_linear_q4_groups_of_different_size(gpu, M, group, ratio):
    """x differs in size between the scale groups of a row, the scales the other way, so that all groups
    count alike: each keeps its own precision."""
    K, N = 1000, 40
    rng = np.random.default_rng(M + group)
    codes, scales, z = (rng.integers(0, 256, (N, K // 2), dtype=np.uint8),
                        (0.01 * (0.2 + rng.random((N, -(-K // group))))).astype(np.float32),
                        rng.integers(0, 16, (N, -(-K // group)), dtype=np.uint8))
    size = ratio ** rng.choice([-0.5, 0.0, 0.5], scales.shape[1])
    scales = (scales / size).astype(np.float32)
    x = (rng.standard_normal((M, K)) * np.repeat(size, group)[:K]).astype(np.float32)
    y = np.zeros((M, N), np.float32)
    gpu.linear_q4(y, x, gpu.Q4Weight(codes, scales, z, K=K, group=group))
    ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), groups=-(-K // group))
    for r in range(M):
        assert (np.abs(y[r] - ref[r]) <= tol[r]).all() and R.rel(y[r], ref[r]) <= 3e-6, (r, R.rel(y[r], ref[r]))
