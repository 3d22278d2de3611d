"""Token-by-token decoding of a Qwen3-shaped language model with 4-bit weights and a 4-bit cache.

A few layers with random weights take a batch of prompts of different lengths, then one token at a
time: fused q/k/v projection, norm and rotation of queries and keys, append to the paged cache,
attention over it, output projection, SiLU-gated MLP, all through ``invision_b200.envg``.  The same
layers in plain torch (fp32, on the values that weights and cache hold) check the result.

    python examples/decode_q4.py [--layers 4] [--batch 4] [--steps 16]
"""
import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from invision_b200 import envg  # noqa: E402

EPS = 1e-6


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


class Layer:
    """One layer: 4-bit weights on the device, its part of the cache, and what the weights stand for."""

    def __init__(self, cfg, rng, group=128):
        d, hd, q, kv, mlp = cfg["hidden"], cfg["head_dim"], cfg["heads"], cfg["kv_heads"], cfg["mlp"]
        self.cfg, self.w, self.plain = cfg, {}, {}
        for name, n, k, layout in (("qkv", (q + 2 * kv) * hd, d, envg.LAYOUT_PLAIN), ("o", d, q * hd, envg.LAYOUT_PLAIN),
                                   ("gate_up", 2 * mlp, d, envg.LAYOUT_GATE_UP), ("down", d, mlp, envg.LAYOUT_PLAIN)):
            codes, scales, zeros = envg.quantize_q4((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32), group)
            self.w[name] = envg.Q4Weight(codes, scales, zeros, K=k, group=group, layout=layout)
            c = np.stack((codes & 15, codes >> 4), -1).reshape(n, -1)[:, :k].astype(np.float32)
            at = np.arange(k) // group
            self.plain[name] = torch.from_numpy((c - zeros[:, at]) * scales[:, at]).cuda()
        vec = lambda n: torch.from_numpy((1 + 0.1 * rng.standard_normal(n)).astype(np.float32)).cuda()  # noqa: E731
        self.norm1, self.norm2, self.qn, self.kn = vec(d), vec(d), vec(hd), vec(hd)
        self.ones = torch.ones(d, device="cuda")
        self.cache = envg.KV4Cache(cfg["pages"], cfg["page"], kv, hd)

    def step(self, x, table, lens, positions, tables, q_len):
        """x [B * q_len, hidden] (changed in place): the newest q_len tokens of each sequence."""
        c, n = self.cfg, x.shape[0]
        hd, q, kv = c["head_dim"], c["heads"], c["kv_heads"]
        qkv = torch.empty((n, (q + 2 * kv) * hd), device="cuda")
        envg.linear_q4(qkv, _norm(x, self.norm1), self.w["qkv"], sync=False)
        qs, ks, vs = qkv[:, : q * hd], qkv[:, q * hd : (q + kv) * hd], qkv[:, (q + kv) * hd :]
        envg.qk_norm_rope(qs, ks, qs, ks, self.qn, self.kn, *tables, q, kv, hd, positions=positions, eps=EPS, sync=False)
        self.cache.append(ks, vs, table, lens, q_len=q_len, sync=False)
        att = torch.empty((n, q * hd), device="cuda")
        envg.attention_kv4(att, qs, self.cache, table, lens, q, q_len=q_len, sync=False)
        envg.linear_q4(x, att, self.w["o"], epilogue=envg.EPI_GATED_RESIDUAL, gate=self.ones, sync=False)
        mid = torch.empty((n, c["mlp"]), device="cuda")
        envg.linear_q4(mid, _norm(x, self.norm2), self.w["gate_up"], sync=False)
        envg.linear_q4(x, mid, self.w["down"], epilogue=envg.EPI_GATED_RESIDUAL, gate=self.ones, sync=False)

    def plain_step(self, x, table, lens, positions, tables, q_len):
        """The same on what weights and cache hold, in plain torch; reads the cache after step()."""
        c = self.cfg
        hd, q, kv, B = c["head_dim"], c["heads"], c["kv_heads"], lens.shape[0]
        cos, sin = (t[positions.long()][:, None] for t in tables)
        qkv = _norm(x, self.norm1) @ self.plain["qkv"].t()

        def turn(y, w):
            a, b = _norm(y.view(x.shape[0], -1, hd), w).chunk(2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        qs = turn(qkv[:, : q * hd], self.qn)
        out = torch.empty((x.shape[0], q, hd), device="cuda")
        for b in range(B):
            n = int(lens[b])
            k, v = (torch.empty((n, kv * hd), device="cuda") for _ in range(2))
            self.cache.read(k, v, table[b : b + 1].contiguous(), lens[b : b + 1], q_len=n)
            k, v = (t.view(n, kv, hd).repeat_interleave(q // kv, 1) for t in (k, v))
            rows = slice(b * q_len, (b + 1) * q_len)
            s = torch.einsum("qhd,nhd->hqn", qs[rows], k) * hd ** -0.5
            hide = torch.arange(n, device="cuda") > (n - q_len + torch.arange(q_len, device="cuda"))[:, None]
            out[rows] = torch.einsum("hqn,nhd->qhd", torch.softmax(s.masked_fill(hide, -torch.inf), -1), v)
        x = x + out.reshape(x.shape[0], -1) @ self.plain["o"].t()
        gate, up = (_norm(x, self.norm2) @ self.plain["gate_up"].t()).chunk(2, 1)
        return x + (torch.nn.functional.silu(gate) * up) @ self.plain["down"].t()


def run(layers=4, batch=4, steps=16, hidden=2560, heads=32, kv_heads=8, head_dim=128, mlp=9728, page=32, prompt=48, check=True,
        seed=0):
    """Decode ``steps`` tokens for each prompt; returns (largest relative error of a step, seconds per step)."""
    envg.init(0)
    rng = np.random.default_rng(seed)
    first = [max(1, prompt - 7 * b) for b in range(batch)]
    per = -(-(prompt + steps) // page)
    cfg = dict(hidden=hidden, heads=heads, kv_heads=kv_heads, head_dim=head_dim, mlp=mlp, page=page, pages=batch * per)
    model = [Layer(cfg, rng) for _ in range(layers)]
    table = torch.from_numpy(rng.permutation(batch * per).astype(np.int32).reshape(batch, per)).cuda()
    angle = np.arange(prompt + steps)[:, None] * 1e6 ** (-np.arange(head_dim // 2) / (head_dim // 2))
    tables = tuple(torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    lens = torch.tensor(first, dtype=torch.int32, device="cuda")
    worst, spent = 0.0, 0.0
    for i in range(steps + 1):
        q_len = prompt if i == 0 else 1  # the prompts first: rows before a short prompt's start are padding
        new = lens[:, None] - q_len + torch.arange(q_len, dtype=torch.int32, device="cuda")
        positions = new.clamp(min=0).reshape(-1).contiguous()
        x = torch.from_numpy(rng.standard_normal((batch * q_len, hidden)).astype(np.float32)).cuda()
        y = x.clone()
        torch.cuda.synchronize()
        began = time.perf_counter()
        for m in model:
            m.step(y, table, lens, positions, tables, q_len)
        envg.sync()
        spent += time.perf_counter() - began if i > 1 else 0.0
        if check:
            # layer by layer on the library's own input, so that only one layer's rounding is seen
            z, w = x, x.clone()
            for m in model:
                m.step(w, table, lens, positions, tables, q_len)
                z = m.plain_step(z, table, lens, positions, tables, q_len)
                real = (new >= 0).reshape(-1)
                worst = max(worst, float((w - z)[real].norm() / z[real].norm()))
                z = w.clone()
        lens += 1
    return worst, spent / max(1, steps - 1)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    err, sec = run(a.layers, a.batch, a.steps)
    print(f"{a.layers} layers, {a.batch} sequences: {1e6 * sec:.0f} us per token step, largest relative error {err:.1e}")
