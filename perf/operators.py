"""The operators of a language-model layer at decode time, as cases to be measured.

* ``linear_q4``      y = epilogue(x . W^T), W held as 4-bit codes with a scale (and zero) per group of a row
* ``qk_norm_rope``   RMS norm of every query and key head and the position rotation, in one pass
* ``kv4_append``     keys and values written to a paged 4-bit cache, and read back as the values it holds
* ``attention_kv4``  attention over that cache: causal, optionally a sliding window plus first tokens (sinks)

``run`` computes them with elementary torch operations in 32 bits (``own`` false) or through
``invision_b200.envg`` (``own`` true).
"""
import math

import numpy as np
import torch

own = False

GROUP = 64  # channels of a cached head that share one scale and one minimum


# ---- cases ------------------------------------------------------------------------------------

def listed():
    return [
        # the key projection of a 2560-wide layer for one new token: a call of a few microseconds
        dict(name="linear_k_1", op="linear_q4", M=1, K=2560, N=1024, group=128, zeros=True, gate_up=False, bias=False),
        # gate and up of that layer's MLP with the SiLU gate, one token
        dict(name="linear_gate_up_1", op="linear_q4", M=1, K=2560, N=19456, group=64, zeros=True, gate_up=True, bias=False),
        # the fused input projection of a 4096-wide block for four rows: the largest weight
        dict(name="linear_fused_in_4", op="linear_q4", M=4, K=4096, N=36864, group=128, zeros=False, gate_up=False, bias=True),
        # the down projection for a batch of 16 sequences, small groups
        dict(name="linear_down_16", op="linear_q4", M=16, K=9728, N=2560, group=32, zeros=True, gate_up=False, bias=False),
        # queries and keys of a batch of 16 tokens being decoded
        dict(name="norm_rope_16", op="qk_norm_rope", T=16, heads=32, kv_heads=8, head_dim=128, interleaved=False),
        # queries and keys of an image block's 4608 rows (4096 image and 512 text), pairs side by side
        dict(name="norm_rope_4608", op="qk_norm_rope", T=4608, heads=24, kv_heads=24, head_dim=128, interleaved=True),
        # one new token for each of 64 sequences
        dict(name="append_64x1", op="kv4_append", B=64, q_len=1, ctx=1500, page=64, kv_heads=8, head_dim=128),
        # a prompt of 4096 tokens
        dict(name="append_1x4096", op="kv4_append", B=1, q_len=4096, ctx=4096, page=64, kv_heads=8, head_dim=128),
        # one sequence at the length of the text encoder's prompts
        dict(name="attn_1x512", op="attention_kv4", B=1, q_len=1, ctx=512, page=16, heads=32, kv_heads=8, head_dim=128, window=0, sinks=0),
        # a batch of 16 long sequences of different lengths
        dict(name="attn_16x16384", op="attention_kv4", B=16, q_len=1, ctx=16384, page=64, heads=32, kv_heads=8, head_dim=128, window=0, sinks=0),
        # 32 sequences that see their last 1024 tokens and the first 4
        dict(name="attn_32x8000_window", op="attention_kv4", B=32, q_len=1, ctx=8000, page=32, heads=32, kv_heads=8, head_dim=128, window=1024, sinks=4),
        # the next 128 tokens of a prompt against what is cached of it
        dict(name="attn_chunk_128", op="attention_kv4", B=1, q_len=128, ctx=8192, page=64, heads=32, kv_heads=8, head_dim=128, window=0, sinks=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear_q4", "linear_q4", "qk_norm_rope", "kv4_append", "attention_kv4", "attention_kv4"])
    if op == "linear_q4":
        gate_up = rng.random() < 0.3
        M, K = _log(rng, 1, 64), _log(rng, 64, 16384)
        N = _log(rng, 16, min(36864, (150_000_000 if M <= 4 else 30_000_000) // K))
        if rng.random() < 0.5:  # the sizes of models are multiples of 64
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        N += N % 2 if gate_up else 0
        return dict(op=op, M=M, K=K, N=N, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, gate_up=gate_up,
                    bias=not gate_up and rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if op == "qk_norm_rope":
        return dict(op=op, T=_log(rng, 1, 4608), heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 96, 128, 256]),
                    interleaved=rng.random() < 0.5)
    head_dim, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if op == "kv4_append":
        B = _log(rng, 1, 64)
        q_len = _log(rng, 1, 4096 // B)
        return dict(op=op, B=B, q_len=q_len, ctx=q_len + rng.randrange(0, 1000), page=page, kv_heads=kv_heads, head_dim=head_dim)
    B = _log(rng, 1, 32)
    q_len = rng.choice([1, 1, 1, 2, 4, _log(rng, 1, max(1, 64 // B))])
    ctx = max(q_len, _log(rng, 1, 16384 * 16 // max(B, 16)))
    window = rng.choice([0, 0, _log(rng, 1, 4096)])
    return dict(op=op, B=B, q_len=q_len, ctx=ctx, page=page, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window,
                sinks=rng.choice([0, 1, 4, 17]) if window else 0)


def _lens(case):
    """Tokens held for each sequence, the new ones among them: the longest first, falling to half."""
    B, ctx = case["B"], case["ctx"]
    return [max(1, ctx - (ctx * b) // (2 * B)) for b in range(B)]


def _visible(case, n):
    """Cached tokens that some new token of a sequence of n sees, and the (new token, cached token) pairs."""
    w, sinks, q = case["window"], case["sinks"], case["q_len"]
    pos = np.arange(max(0, n - q), n, dtype=np.int64)
    if not w:
        return n, int((pos + 1).sum())
    seen = np.minimum(pos + 1, w) + np.minimum(np.maximum(pos + 1 - w, 0), sinks)
    first = max(0, int(pos[0]) + 1 - w)
    return n - first + min(first, sinks), int(seen.sum())


def work(case):
    op = case["op"]
    if op == "linear_q4":
        M, K, N = case["M"], case["K"], case["N"]
        groups = -(-K // case["group"])
        n_out = N // 2 if case["gate_up"] else N
        held = N * ((K + 1) // 2) + N * groups * (5 if case["zeros"] else 4)
        return dict(bytes=held + 4 * M * K + 4 * M * n_out + (4 * N if case["bias"] else 0), flops=2 * M * N * K)
    hd = case["head_dim"]
    if op == "qk_norm_rope":
        n = case["T"] * (case["heads"] + case["kv_heads"]) * hd
        return dict(bytes=8 * n + 4 * case["T"] * (hd + 1) + 8 * hd, flops=7 * n)
    held = case["kv_heads"] * (hd + 8 * (hd // GROUP))  # bytes of one token's keys and values in the cache
    if op == "kv4_append":
        n = case["B"] * case["q_len"]
        new = sum(min(case["q_len"], v) for v in _lens(case))
        return dict(bytes=2 * 8 * n * case["kv_heads"] * hd + 2 * new * held, flops=16 * n * case["kv_heads"] * hd)
    tokens, pairs = (sum(v) for v in zip(*[_visible(case, n) for n in _lens(case)]))
    rows = case["B"] * case["q_len"]
    return dict(bytes=tokens * held + 8 * rows * case["heads"] * hd, flops=4 * pairs * case["heads"] * hd)


# ---- inputs -----------------------------------------------------------------------------------

def _kv_quantize(x, fifteen):
    """Codes, scale and minimum of groups of the last dimension: [..., GROUP] -> uint8, half, half."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = lo.clamp(-65504.0, 65504.0).half()
    s = ((hi - lo) / fifteen).clamp(max=65504.0).half()
    c = torch.round((x - m.float()) / s.float()).clamp(0.0, 15.0)
    return torch.where(s > 0, c, torch.zeros_like(c)).to(torch.uint8), s, m


def _tables(case, gen, dev):
    """A page table in random order with a few pages to spare: (table, lengths, pages)."""
    per = -(-case["ctx"] // case["page"])
    pages = case["B"] * per + 3
    order = torch.randperm(pages, generator=gen, device=dev)[: case["B"] * per]
    return order.view(case["B"], per).to(torch.int32), torch.tensor(_lens(case), dtype=torch.int32, device=dev), pages


def _keys(shape, gen, dev):
    """Keys as rotation leaves them: some channels far from zero and wider than others."""
    x = torch.randn(shape, generator=gen, device=dev)
    hd = shape[-1]
    x *= 0.5 + 1.5 * torch.rand(shape[-2:], generator=gen, device=dev)
    return x.add_(2.0 * (torch.rand((shape[-2], hd), generator=gen, device=dev) < 0.05))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    st = dict(case=case, fifteen=torch.full((1,), 15.0, device=dev))
    if own:
        from invision_b200 import envg

        envg.init(0)
        st["envg"] = envg
    op = case["op"]
    if op == "linear_q4":
        M, K, N, g = case["M"], case["K"], case["N"], case["group"]
        groups = -(-K // g)
        st["codes"] = torch.randint(0, 256, (N, (K + 1) // 2), generator=gen, device=dev, dtype=torch.uint8)
        st["scales"] = 0.005 * (0.5 + torch.rand((N, groups), generator=gen, device=dev))
        st["zeros"] = torch.randint(5, 11, (N, groups), generator=gen, device=dev, dtype=torch.uint8) if case["zeros"] else None
        st["x"] = torch.randn((M, K), generator=gen, device=dev)
        st["bias"] = 0.01 * torch.randn((N,), generator=gen, device=dev) if case["bias"] else None
        if own:
            layout = envg.LAYOUT_GATE_UP if case["gate_up"] else envg.LAYOUT_PLAIN
            st["w"] = envg.Q4Weight(st["codes"], st["scales"], st["zeros"], K=K, group=g, layout=layout)
            st["y"] = torch.empty((M, N // 2 if case["gate_up"] else N), device=dev)
        return st
    hd, kvh = case["head_dim"], case["kv_heads"]
    if op == "qk_norm_rope":
        T, H = case["T"], case["heads"]
        st["q"] = torch.randn((T, H * hd), generator=gen, device=dev)
        st["k"] = torch.randn((T, kvh * hd), generator=gen, device=dev)
        st["wq"] = 1.0 + 0.1 * torch.randn((hd,), generator=gen, device=dev)
        st["wk"] = 1.0 + 0.1 * torch.randn((hd,), generator=gen, device=dev)
        angle = torch.arange(8192, device=dev)[:, None] * (1e6 ** (-torch.arange(hd // 2, device=dev) / (hd // 2)))
        st["cos"], st["sin"] = torch.cos(angle), torch.sin(angle)
        first = torch.randint(0, 8192 - T, (1,), generator=gen, device=dev)
        st["pos"] = (first + torch.arange(T, device=dev)).to(torch.int32)
        if own:
            st["q_out"], st["k_out"] = torch.empty_like(st["q"]), torch.empty_like(st["k"])
        return st
    B, q_len = case["B"], case["q_len"]
    st["table"], st["lens"], pages = _tables(case, gen, dev)
    if op == "kv4_append":
        st["k"] = _keys((B * q_len, kvh, hd), gen, dev).view(B * q_len, kvh * hd)
        st["v"] = torch.randn((B * q_len, kvh * hd), generator=gen, device=dev)
        if own:
            st["cache"] = envg.KV4Cache(pages, case["page"], kvh, hd)
            st["k_out"], st["v_out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
        return st
    st["q"] = torch.randn((B * q_len, case["heads"] * hd), generator=gen, device=dev)
    k = _keys((pages, case["page"], kvh, hd), gen, dev)
    v = torch.randn((pages, case["page"], kvh, hd), generator=gen, device=dev)
    if own:
        st["cache"] = envg.KV4Cache(pages, case["page"], kvh, hd)
        st["out"] = torch.empty_like(st["q"])
        held = st["table"].shape[1] * case["page"]
        rows = [t[st["table"].long()].view(B * held, kvh * hd) for t in (k, v)]
        st["cache"].append(*rows, st["table"], torch.full_like(st["lens"], held), q_len=held)
    for name, t in (("k", k), ("v", v)):  # the cache's contents: two codes to a byte, scale and minimum per group
        c, s, m = _kv_quantize(t.view(pages, case["page"], kvh, hd // GROUP, GROUP), st["fifteen"])
        c = c.view(pages, case["page"], kvh, hd)
        st[name] = (c[..., 0::2] | (c[..., 1::2] << 4), s, m)
    return st


# ---- one pass ---------------------------------------------------------------------------------

def run(st):
    return _own_run(st) if own else _plain_run(st)


def _own_run(st):
    case, envg = st["case"], st["envg"]
    op = case["op"]
    if op == "linear_q4":
        envg.linear_q4(st["y"], st["x"], st["w"], bias=st["bias"], sync=False)
        return st["y"]
    if op == "qk_norm_rope":
        envg.qk_norm_rope(st["q_out"], st["k_out"], st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"],
                          case["heads"], case["kv_heads"], case["head_dim"], positions=st["pos"],
                          interleaved=case["interleaved"], sync=False)
        return st["q_out"], st["k_out"]
    if op == "kv4_append":
        st["cache"].append(st["k"], st["v"], st["table"], st["lens"], q_len=case["q_len"], sync=False)
        st["cache"].read(st["k_out"], st["v_out"], st["table"], st["lens"], q_len=case["q_len"], sync=False)
        return st["k_out"], st["v_out"]
    envg.attention_kv4(st["out"], st["q"], st["cache"], st["table"], st["lens"], case["heads"], q_len=case["q_len"],
                       max_ctx=case["ctx"], window=case["window"], sinks=case["sinks"], sync=False)
    return st["out"]


def _plain_run(st):
    return dict(linear_q4=_plain_linear, qk_norm_rope=_plain_norm_rope, kv4_append=_plain_append,
                attention_kv4=_plain_attention)[st["case"]["op"]](st)


def _plain_linear(st):
    case = st["case"]
    K, codes = case["K"], st["codes"]
    c = torch.stack((codes & 15, codes >> 4), dim=-1).view(codes.shape[0], -1)[:, :K]
    at = torch.arange(K, device=codes.device) // case["group"]
    z = st["zeros"].float()[:, at] if st["zeros"] is not None else 8.0
    y = st["x"] @ ((c.float() - z) * st["scales"][:, at]).t()
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["gate_up"]:
        gate, up = y.chunk(2, dim=1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y


def _plain_norm_rope(st):
    case = st["case"]
    T, hd = case["T"], case["head_dim"]
    at = st["pos"].long()
    cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]

    def one(x, w):
        x = x.view(T, -1, hd)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        if case["interleaved"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).view(T, -1)
        a, b = x[..., : hd // 2], x[..., hd // 2 :]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).view(T, -1)

    return one(st["q"], st["wq"]), one(st["k"], st["wk"])


def _plain_append(st):
    case = st["case"]
    B, q_len, kvh, hd, page = case["B"], case["q_len"], case["kv_heads"], case["head_dim"], case["page"]
    # tokens of a sequence stand at its end; rows before its first token belong to none
    pos = st["lens"].long()[:, None] - q_len + torch.arange(q_len, device=st["k"].device)
    slot = st["table"].long().gather(1, pos.clamp(min=0) // page) * page + pos.clamp(min=0) % page
    pages = case["B"] * st["table"].shape[1] + 3

    def one(x):
        c, s, m = _kv_quantize(x.view(B * q_len, kvh, hd // GROUP, GROUP), st["fifteen"])
        c = c.view(B * q_len, kvh, hd)
        there = (pos >= 0).view(-1)
        held = torch.zeros((pages * page, kvh, hd // 2), dtype=torch.uint8, device=x.device)
        held_s, held_m = (torch.zeros((pages * page, kvh, hd // GROUP, 1), dtype=torch.half, device=x.device) for _ in range(2))
        at = slot.view(-1)[there]
        held[at], held_s[at], held_m[at] = (c[..., 0::2] | (c[..., 1::2] << 4))[there], s[there], m[there]
        at = slot.view(-1)
        c = torch.stack((held[at] & 15, held[at] >> 4), dim=-1).view(B * q_len, kvh, hd // GROUP, GROUP)
        y = held_m[at].float() + held_s[at].float() * c.float()
        return torch.where(there[:, None], y.view(B * q_len, kvh * hd), torch.zeros((), device=x.device))

    return one(st["k"]), one(st["v"])


def _mask(case, lens, L, device):
    """[B, q_len, L]: which cached tokens each new token sees."""
    pos = lens[:, None] - case["q_len"] + torch.arange(case["q_len"], device=device)
    j = torch.arange(L, device=device)
    see = j <= pos[..., None]
    if case["window"]:
        see &= (j > pos[..., None] - case["window"]) | (j < case["sinks"])
    return see


def _plain_attention(st):
    case = st["case"]
    B, q_len, H, kvh, hd = case["B"], case["q_len"], case["heads"], case["kv_heads"], case["head_dim"]
    table = st["table"].long()

    def values(held):
        codes, s, m = (t[table] for t in held)
        c = torch.stack((codes & 15, codes >> 4), dim=-1).view(*codes.shape[:4], hd // GROUP, GROUP)
        return (m.float() + s.float() * c.float()).view(B, -1, kvh, hd).transpose(1, 2)  # [B, kvh, L, hd]

    k, v = values(st["k"]), values(st["v"])
    q = st["q"].view(B, q_len, kvh, H // kvh, hd).permute(0, 2, 3, 1, 4).reshape(B, kvh, -1, hd)
    see = _mask(case, st["lens"].long(), k.shape[2], q.device)[:, None].repeat(1, H // kvh, 1, 1).view(B, 1, -1, k.shape[2])
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    x = torch.where(see, x, torch.full((), -math.inf, device=q.device))
    top = x.amax(-1, keepdim=True)
    p = torch.where(see, torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros_like(x))
    total = p.sum(-1, keepdim=True)
    y = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return y.view(B, kvh, H // kvh, q_len, hd).permute(0, 3, 1, 2, 4).reshape(B * q_len, H * hd)


# ---- the operators in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "linear_q4":
        N, K, g = case["N"], case["K"], case["group"]
        if N * K > 160_000_000:
            return None
        w = torch.empty((N, 2 * st["codes"].shape[1]), dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = st["codes"].remainder(16), torch.div(st["codes"], 16, rounding_mode="floor")
        w = w[:, :K]
        w -= 8.0 if st["zeros"] is None else st["zeros"].double().repeat_interleave(g, 1)[:, :K]
        w *= st["scales"].double().repeat_interleave(g, 1)[:, :K]
        y = torch.einsum("mk,nk->mn", st["x"].double(), w)
        y += 0.0 if st["bias"] is None else st["bias"].double()
        if case["gate_up"]:
            y = y[:, : N // 2] * torch.sigmoid(y[:, : N // 2]) * y[:, N // 2 :]
        return y
    hd = case["head_dim"]
    if op == "qk_norm_rope":
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, None]
        got = []
        for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
            x = x.double().view(case["T"], -1, hd)
            x = x / ((x * x).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * w.double()
            x = x.unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
            axis = -1 if case["interleaved"] else -2
            z = torch.complex(*(t.contiguous() for t in x.unbind(axis))) * turn
            got.append(torch.stack((z.real, z.imag), axis).reshape(case["T"], -1))
        return tuple(got)
    if op == "kv4_append":
        lens = np.repeat(np.asarray(_lens(case)), case["q_len"])
        there = lens - case["q_len"] + np.tile(np.arange(case["q_len"]), case["B"]) >= 0
        got = []
        for x in (st["k"], st["v"]):
            x = x.double().cpu().numpy().reshape(len(there), -1, GROUP)
            least, most = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
            m = least.astype(np.float16).astype(np.float64)
            s = ((most - least) / 15.0).astype(np.float16).astype(np.float64)
            c = np.clip(np.rint(np.divide(x - m, s, out=np.zeros_like(x), where=s > 0)), 0, 15)
            got.append(torch.from_numpy(((m + s * c) * there[:, None, None]).reshape(len(there), -1)))
        return tuple(got)
    # attention, a sequence at a time: the tokens held, then a softmax over those that are seen
    H, kvh, q_len = case["heads"], case["kv_heads"], case["q_len"]
    out = torch.zeros((case["B"], q_len, H, hd), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        kv = []
        for codes, s, m in (st["k"], st["v"]):
            at = st["table"][b].long()
            codes, s, m = (t[at].flatten(0, 1)[:n].double() for t in (codes, s, m))
            high = torch.floor(codes / 16)
            c = torch.stack((codes - 16 * high, high), -1).reshape(n, kvh, hd // GROUP, GROUP)
            kv.append((c * s + m).reshape(n, kvh, hd).repeat_interleave(H // kvh, 1))
        q = st["q"].double().view(case["B"], q_len, H, hd)[b]
        x = torch.einsum("qhd,nhd->hqn", q, kv[0]) / math.sqrt(hd)
        pos = n - q_len + torch.arange(q_len, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = j > pos
        if case["window"]:
            hidden = hidden | ((pos - j >= case["window"]) & (j >= case["sinks"]))
        p = torch.softmax(x.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
        out[b] = torch.einsum("hqn,nhd->qhd", p, kv[1])
    return out.view(case["B"] * q_len, H * hd)
