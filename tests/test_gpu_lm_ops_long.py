"""GPU: the language-model decode operators at sizes where a CTA or a warp goes through its loops
several times: rounds of row tiles of the 4-bit linear, batches of looked-up pages of the attention."""
import numpy as np
import pytest

from tests import lm_ref as R
from tests.test_gpu_lm_ops import REL, _close
from tests.test_gpu_lm_ops_accuracy import REL_GROUP

pytestmark = pytest.mark.gpu


# The linear gives each cluster of 1, 2, 4 or 8 CTAs a run of row tiles and takes 32 of them at a time.
@pytest.mark.parametrize("M,K,N,group,gate_up", [
    (64, 256, 20000, 64, False),   # 34 tiles to a CTA: the second round is two tiles
    (200, 1000, 8200, 64, True),   # 47 to a CTA, thirteen launch rows
    (1, 256, 90000, 128, False),   # one row, 39 to a CTA
    (3, 300, 80000, 64, False),    # three rows, 34 to a CTA, a block that K ends inside
    (300, 2100, 2500, 128, False),  # clusters of two, 53 tiles
    (40, 3000, 9000, 32, False),   # clusters of four, 47 tiles
    (70, 2049, 9002, 32, True),    # clusters of two, odd sizes, pairs of rows
    (300, 4096, 6000, 32, False),  # one cluster of four for each launch row, 375 tiles
    (64, 9728, 5000, 128, False),  # clusters of eight, 79 tiles
    (1, 57344, 70, 32, False),     # the longest rows: one, four, eight (as twice four) and nine of them
    (4, 57344, 40, 32, False),
    (8, 57344, 33, 64, False),
    (9, 57344, 40, 128, True),
])
def test_linear_q4_in_rounds(gpu, M, K, N, group, gate_up):
    rng = np.random.default_rng(M + N)
    groups = -(-K // group)
    codes = rng.integers(0, 256, (N, (K + 1) // 2), dtype=np.uint8)
    scales = (0.01 * (0.2 + rng.random((N, groups)))).astype(np.float32)
    z = rng.integers(0, 16, (N, groups), dtype=np.uint8)
    x = rng.standard_normal((M, K)).astype(np.float32)
    W = gpu.Q4Weight(codes, scales, z, K=K, group=group, layout=gpu.LAYOUT_GATE_UP if gate_up else gpu.LAYOUT_PLAIN)
    y = np.full((M, N // 2 if gate_up else N), np.nan, np.float32)
    gpu.linear_q4(y, x, W)
    ref, tol = R.linear(x, R.q4_weight(codes, scales, z, K, group), gate_up=gate_up, groups=groups)
    if gate_up:
        assert np.isfinite(y).all() and (np.abs(y - ref) - tol).max() <= 0 and R.rel(y, ref) <= 2 * REL
    else:
        _close(y, ref, tol, f"{M}x{K}x{N}")


def _sequences(rng, n, B, page, spare):
    """B sequences of up to n tokens over the same pages, each in an order of its own: (table, lens)."""
    per = -(-n // page)
    table = np.stack([rng.permutation(per + spare)[:per] for _ in range(B)]).astype(np.int32)
    return table, np.array([n - (17 * b) % (n // 3) for b in range(B)], np.int32)


def _pages(gpu, rng, pages, page, KVH, hd):
    """A full cache, and the values it holds: [pages, page, KVH, hd]."""
    c = gpu.KV4Cache(pages, page, KVH, hd)
    k = rng.standard_normal((pages * page, KVH, hd)).astype(np.float32)
    v = rng.standard_normal((pages * page, KVH, hd)).astype(np.float32)
    n = pages * page
    c.append(k.reshape(n, -1), v.reshape(n, -1), np.arange(pages, dtype=np.int32)[None], np.array([n], np.int32), q_len=n)
    return c, R.kv_hold(k).reshape(pages, page, KVH, hd), R.kv_hold(v).reshape(pages, page, KVH, hd)


# A warp takes units of 32 tokens and looks the pages of 16 units up at a time.
@pytest.mark.parametrize("n,B,q_len,H,KVH,hd,page,window", [
    (34000, 1, 1, 4, 1, 128, 16, 0),      # 33 units a warp in a cluster of eight
    (34000, 1, 1, 8, 1, 64, 64, 0),       # eight rows at a time
    (40000, 1, 1, 2, 1, 128, 32, 39000),
    (9000, 40, 1, 8, 8, 64, 16, 0),       # 35 units a warp, two CTAs to a group
    (5000, 40, 1, 64, 8, 64, 48, 0),
    (20000, 1, 64, 8, 2, 128, 64, 0),     # a chunk far into a long prompt
    (17000, 2, 5, 6, 2, 64, 128, 0),
])
def test_attention_kv4_long(gpu, n, B, q_len, H, KVH, hd, page, window):
    rng = np.random.default_rng(n + H)
    spare = 3
    table, lens = _sequences(rng, n, B, page, spare)
    c, k, v = _pages(gpu, rng, table.shape[1] + spare, page, KVH, hd)
    q = rng.standard_normal((B * q_len, H * hd)).astype(np.float32)
    out = np.full_like(q, np.nan)
    gpu.attention_kv4(out, q, c, table, lens, H, q_len=q_len, max_ctx=int(lens.max()), window=window, sinks=5)
    for b in range(B) if B <= 4 else (0, 1, B // 2, B - 1):
        rows = slice(b * q_len, (b + 1) * q_len)
        kk, vv = (t[table[b]].reshape(-1, KVH, hd)[: lens[b]] for t in (k, v))
        ref = R.attention_exact(q[rows].reshape(q_len, H, hd), kk, vv, lens[b] - q_len + np.arange(q_len), window, 5, hd ** -0.5)
        got = out[rows].reshape(q_len, H, hd)
        assert np.isfinite(got).all() and R.rel(got, ref) <= REL_GROUP, (b, R.rel(got, ref))


@pytest.mark.parametrize("H", [4, 8])
def test_attention_kv4_missing_pages_of_a_long_sequence(gpu, H):
    """Pages that the table does not name, in every batch of looked-up pages: their tokens are left out,
    all others are seen, and the call reports it."""
    import torch

    n, page, hd = 36000, 16, 64
    rng = np.random.default_rng(H)
    table, lens = _sequences(rng, n, 1, page, 3)
    c, k, v = _pages(gpu, rng, table.shape[1] + 3, page, 1, hd)
    gone = np.array([0, 700, 1023, 1024, 1025, 2100, table.shape[1] - 1])
    bad = table.copy()
    bad[0, gone] = [-1, 1 << 30, -5, table.shape[1] + 3, -1, -(1 << 31), -1]
    q = rng.standard_normal((1, H * hd)).astype(np.float32)
    out, dev = torch.full((1, H * hd), float("nan"), device="cuda"), lambda a: torch.from_numpy(a).cuda()
    with pytest.raises(gpu.EnvgError, match="page"):
        gpu.attention_kv4(out, dev(q), c, dev(bad), dev(lens), H, max_ctx=n)
    keep = np.ones(n, bool)
    for i in gone:
        keep[i * page : (i + 1) * page] = False
    kk, vv = (t[table[0]].reshape(-1, 1, hd)[:n][keep] for t in (k, v))
    ref = R.attention_exact(q.reshape(1, H, hd), kk, vv, [n], 0, 0, hd ** -0.5)
    assert R.rel(out.cpu().numpy().reshape(1, H, hd), ref) <= REL_GROUP
