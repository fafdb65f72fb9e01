"""Performance cases of what a decoder layer's mixers do between their projections, through the package's public calls.

Families (`kind`), each over the sizes a serving engine meets:
  conv    the short causal convolution of an SSM layer over packed prompts or single tokens, with the rows'
          last inputs kept, StateCache.conv;
  scan    the selective state space scan behind it, over packed prompts (in part continued ones) or single
          tokens, with the rows' states kept, StateCache.scan;
  rotate  norms of the query and key heads and their rotation in one pass, rotary.rotate;
  append  the same for a step whose keys and values go into one layer's pages, KVCache.append_rotated.

Inputs of a scan are what a convolution with SiLU gives; steps and decays are spread as such models begin
their training: softplus(bias) over the logarithm of 0.001..0.1, -A over 1..16. Lengths of a batch are spread
over the logarithm of their range, the same for every seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch
import torch.nn.functional as F

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
WIDTH = 4   # taps of the convolution
CHUNK = 64  # tokens of a block of the plain scan
EPS = 1e-6  # of the norms


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # A full decode batch through an SSM layer's convolution (the decoder's 10240 channels).
        dict(name="conv_bf16_decode_64", kind="conv", dtype="bf16", lens="", batch=64, channels=10240, fresh=False),
        # A ragged batch of prompts, the lengths a scheduler packs into one step; every other one begins.
        dict(name="conv_f16_ragged", kind="conv", dtype="f16", lens="1008,333,64,1,511,129", batch=6, channels=10240, fresh=True),
        # One chat, one token: the decode step where latency counts (48 heads of 128, states of 128).
        dict(name="scan_f16_decode_1", kind="scan", dtype="f16", lens="", batch=1, heads=48, groups=16, dim=128, state=128, gate=True,
             fresh=False),
        # A full decode batch: the largest streams of states.
        dict(name="scan_bf16_decode_64", kind="scan", dtype="bf16", lens="", batch=64, heads=48, groups=16, dim=128, state=128, gate=True,
             fresh=False),
        # A split-fuse step's 64-token prompt chunk, continued.
        dict(name="scan_bf16_chunk_64", kind="scan", dtype="bf16", lens="64", batch=1, heads=48, groups=16, dim=128, state=128, gate=True,
             fresh=False),
        # A ragged batch of prompts on heads of 64 with states of 128 in one group; every other one begins.
        dict(name="scan_f16_ragged", kind="scan", dtype="f16", lens="1008,333,64,1,511,129", batch=6, heads=80, groups=1, dim=64, state=128,
             gate=False, fresh=True),
        # One long prompt: the largest prefill.
        dict(name="scan_bf16_8192", kind="scan", dtype="bf16", lens="8192", batch=1, heads=48, groups=16, dim=128, state=128, gate=True,
             fresh=True),
        # Sixteen single tokens at far positions, whole heads of 128 in pairs of neighbours, no norms.
        dict(name="rotate_f16_16_far", kind="rotate", dtype="f16", tokens=16, seqs=16, first=1000000, heads=48, kv_heads=8, dim=128, rot=128,
             layout="interleaved", norm=False, base=500000.0, factor=8.0),
        # A prompt of the decoder's heads (24 and 4 of 256, a quarter of each rotated), with norms, scaled for long contexts.
        dict(name="rotate_bf16_4096", kind="rotate", dtype="bf16", tokens=4096, seqs=1, first=0, heads=24, kv_heads=4, dim=256, rot=64,
             layout="half", norm=True, base=1000000.0, factor=4.0),
        # A split-fuse step's 80 single tokens into one layer's pages, the decoder's heads.
        dict(name="append_bf16_80", kind="append", dtype="bf16", batch=80, tokens=1, lo=80, hi=4096, heads=24, kv_heads=4, dim=256, rot=64,
             layout="half", norm=True, base=1000000.0, factor=1.0, page=64),
        # The rest of a prompt on top of what is cached, whole heads of 128.
        dict(name="append_f16_1008", kind="append", dtype="f16", batch=1, tokens=1008, lo=7008, hi=7008, heads=48, kv_heads=8, dim=128,
             rot=128, layout="half", norm=False, base=500000.0, factor=1.0, page=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw(rng):
    kind = rng.choice(["conv", "conv", "scan", "scan", "scan", "scan", "rotate", "rotate", "append", "append"])
    dtype = rng.choice(["f16", "bf16"])
    if kind in ("conv", "scan"):
        if rng.random() < 0.4:
            lens, batch = "", _log_int(rng, 1, 64)
        else:
            batch = rng.choice([1, 1, rng.randint(2, 8)])
            top = _log_int(rng, 4, 8192)
            lens = ",".join(str(_log_int(rng, 1, top)) for _ in range(batch)) if batch > 1 else str(top)
        c = dict(kind=kind, dtype=dtype, lens=lens, batch=batch, fresh=bool(lens) and rng.random() < 0.5)
        if kind == "conv":
            return dict(c, channels=8 * _log_int(rng, 64, 1280))
        H, G, P, N = rng.choice([(48, 16, 128, 128), (48, 16, 128, 128), (80, 1, 64, 128), (64, 8, 64, 128), (32, 2, 64, 64), (24, 1, 64, 256),
                                 (16, 16, 128, 64), (32, 1, 128, 256)])
        return dict(c, heads=H, groups=G, dim=P, state=N, gate=rng.random() < 0.5)
    H, Hkv, D = rng.choice([(48, 8, 128), (24, 4, 256), (32, 8, 128), (16, 16, 64), (32, 4, 64), (40, 8, 128), (8, 1, 128), (16, 2, 256)])
    c = dict(kind=kind, dtype=dtype, heads=H, kv_heads=Hkv, dim=D, rot=rng.choice([16, 32, D // 4, D // 2, D, D]),
             layout=rng.choice(["half", "interleaved"]), norm=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0, 1000000.0]),
             factor=rng.choice([1.0, 1.0, 4.0, 40.0]))
    if kind == "rotate":
        tokens = _log_int(rng, 1, 4096)
        return dict(c, tokens=tokens, seqs=rng.randint(1, min(tokens, 8)), first=rng.choice([0, 0, _log_int(rng, 1, 1000000)]))
    tokens = rng.choice([1, 1, 64, _log_int(rng, 1, 1024)])
    hi = max(tokens, _log_int(rng, 64, 8192))
    return dict(c, batch=_log_int(rng, 1, 128 if tokens == 1 else 4), tokens=tokens, lo=max(tokens, _log_int(rng, 1, hi)), hi=hi,
                page=rng.choice([16, 32, 64, 128]))


def _cost(case):
    """What the plain form of a case costs, by the elements of its padded inputs and states."""
    if case["kind"] == "scan":
        n = _seq_lens(case)
        blocks = 1 if not case["lens"] else len(n) * -(-max(n) // CHUNK)
        return blocks * (case["batch"] if not case["lens"] else 1) * case["heads"] * case["dim"] * case["state"]
    if case["kind"] == "conv":
        return len(_seq_lens(case)) * max(_seq_lens(case)) * case["channels"]
    return work(case)["bytes"]


def _load(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 4e14


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, odd ones among them; none with more work,
    or a larger plain form, than the listed ones of its kind."""
    while True:
        c = _draw(rng)
        peers = [x for x in listed() if x["kind"] == c["kind"]]
        if _load(c) <= max(_load(x) for x in peers) and _cost(c) <= max(_cost(x) for x in peers):
            return c


# ---------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n lengths over the logarithm of lo..hi, both ends among them, in a scattered order."""
    u = [(i * 0.6180339887498949) % 1.0 for i in range(n)]
    got = [int(round(lo * (hi / lo) ** x)) for x in u]
    got[-1] = hi
    return [min(max(x, lo), hi) for x in got]


def _seq_lens(case):
    """New tokens of each sequence of a convolution or a scan."""
    return [int(x) for x in case["lens"].split(",")] if case["lens"] else [1] * case["batch"]


def _frequencies(case):
    """(angle of one position for each pair in 64 bits, factor of cosine and sine): base^(-2 i / R), where factor > 1
    stretched by parts for contexts longer than 4096: slow pairs take positions / factor, fast ones stay, a ramp between them."""
    R, base, s = case["rot"], case["base"], case["factor"]
    i = np.arange(R // 2, dtype=np.float64)
    f = base ** (-2.0 * i / R)
    if s == 1.0:
        return f, 1.0
    at = lambda turns: R * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), R - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
    return f / s * ramp + f * (1.0 - ramp), 0.1 * math.log(s) + 1.0


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    k, dt = case["kind"], DTYPES[case["dtype"]]
    f32 = torch.float32
    randn = lambda *shape, dtype=dt: torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, device="cuda", generator=gen)  # noqa: E731
    s = {"case": case}
    if k in ("conv", "scan"):
        lens = _seq_lens(case)
        T, B = sum(lens), len(lens)
        rows = B + 2  # the pool holds others beside the call's
        s["rows"] = _i32(rng.permutation(rows)[:B])
        s["max_len"] = max(lens)
        if case["lens"]:
            s["cu"] = _i32(np.concatenate([[0], np.cumsum(lens)]))
        if case["fresh"]:
            s["held"] = _i32(100 * (np.arange(B) % 2))  # every other sequence begins with the call
    if k == "conv":
        C = case["channels"]
        # The projection's output, the gate beside it.
        s["x"] = randn(T, C + 512)[:, 512:]
        s["weight"], s["bias"] = randn(C, WIDTH, dtype=f32) * 0.5, randn(C, dtype=f32) * 0.1
        s["conv"] = randn(1, rows, WIDTH - 1, C)
        return s
    if k == "scan":
        H, G, P, N = case["heads"], case["groups"], case["dim"], case["state"]
        xbc = F.silu(randn(T, H * P + 2 * G * N))  # one row a token: x, B, C, as the convolution leaves them
        s["x"] = xbc[:, :H * P].view(T, H, P)
        s["B"], s["C"] = (xbc[:, H * P + j * G * N:][:, :G * N].view(T, G, N) for j in (0, 1))
        s["z"] = randn(T, H, P) if case["gate"] else None
        s["dt"] = randn(T, H) * 0.5
        step = torch.exp(rand(H) * math.log(100.0) + math.log(0.001))
        s["dt_bias"] = torch.log(torch.expm1(step))  # softplus of it is the step
        s["A"], s["D"] = -(1 + 15 * rand(H)), 1 + 0.1 * randn(H, dtype=f32)
        s["ssm"] = 0.02 * randn(1, rows, H, P, N, dtype=f32)  # about what such inputs leave
        return s
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    turns, s["mscale"] = _frequencies(case)
    s["angles"] = torch.from_numpy(turns).cuda()
    if case["norm"]:
        s["q_weight"], s["k_weight"] = 1 + 0.1 * randn(D, dtype=f32), 1 + 0.1 * randn(D, dtype=f32)
    if k == "rotate":
        T, n = case["tokens"], case["seqs"]
        cu = np.concatenate([[0], np.sort(rng.permutation(T - 1)[:n - 1] + 1), [T]])
        at = np.arange(T) - np.repeat(cu[:-1], np.diff(cu))
        s["positions"] = _i32(case["first"] + at + 17 * np.repeat(np.arange(n), np.diff(cu)))
    else:
        B, m, page = case["batch"], case["tokens"], case["page"]
        lens = np.array(_spread(B, case["lo"], case["hi"]))
        T, used = B * m, -(-lens // page)
        pages = int(used.sum()) + 3
        order = rng.permutation(pages)
        table = np.full((B, int(used.max()) + 1), -1, np.int64)
        at = np.concatenate([[0], np.cumsum(used)])
        for i in range(B):
            table[i, :used[i]] = order[at[i]:at[i + 1]]
        s["table"], s["lens"], s["refs"] = _i32(table), _i32(lens), _i32(np.bincount(table[table >= 0], minlength=pages))
        s["k_pool"], s["v_pool"] = randn(1, pages, Hkv, page, D), randn(1, pages, Hkv, page, D)
        s["rows"] = torch.arange(B, dtype=torch.int32, device="cuda")
        if m > 1:
            s["cu"] = torch.arange(B + 1, dtype=torch.int32, device="cuda") * m
        s["v"] = randn(T, Hkv, D)
    # The projections' outputs: q with its gate beside it, k.
    s["q"] = randn(T, 2 * H * D)[:, :H * D].view(T, H, D)
    s["k"] = randn(T, Hkv, D)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s, s["case"]["kind"])


def _run_own(s, k):
    if k in ("conv", "scan"):
        from nebula_amd import ssm

        if "cache" not in s:  # the handle that a program makes once
            s["cache"] = ssm.StateCache(conv=s.get("conv"), ssm=s.get("ssm"))
        c = s["cache"]
        if k == "conv":
            return [c.conv(0, s["x"], s["weight"], s["rows"], s.get("cu"), bias=s["bias"], held=s.get("held")), s["conv"]]
        return [c.scan(0, s["x"], s["dt"], s["A"], s["B"], s["C"], s["rows"], s.get("cu"), D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                       held=s.get("held"), max_len=s["max_len"]), s["ssm"]]
    from nebula_amd import attn, rotary

    case = s["case"]
    if "rotary" not in s:
        scaling = None if case["factor"] == 1.0 else rotary.Stretch(case["factor"], 4096)
        s["rotary"] = rotary.Rotary(case["rot"], base=case["base"], layout=case["layout"], scaling=scaling)
        if k == "append":
            s["cache"] = attn.KVCache(s["k_pool"], s["v_pool"], s["table"], s["lens"], s["refs"])
    if k == "rotate":
        return rotary.rotate(s["q"], s["k"], s["rotary"], s["positions"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), eps=EPS)
    q = s["cache"].append_rotated(0, s["rotary"], s["q"], s["k"], s["v"], s["rows"], s.get("cu"), q_weight=s.get("q_weight"),
                                  k_weight=s.get("k_weight"), eps=EPS)
    return [q, s["k_pool"], s["v_pool"]]


def _run_plain(s, k):
    if k == "conv":
        return _conv_plain(s)
    if k == "scan":
        return _step_plain(s) if "cu" not in s else _scan_plain(s)
    if k == "rotate":
        return (_rotated(s, s["q"], s["positions"], s.get("q_weight")), _rotated(s, s["k"], s["positions"], s.get("k_weight")))
    T, m, lens = s["case"]["page"], s["case"]["tokens"], s["lens"].long()
    at = (lens[:, None] - m + torch.arange(m, device=lens.device)).reshape(-1)
    row = torch.arange(len(lens), device=lens.device).repeat_interleave(m)
    page = s["table"][row, at // T].long()
    s["k_pool"][0].transpose(1, 2)[page, at % T] = _rotated(s, s["k"], at, s.get("k_weight"))
    s["v_pool"][0].transpose(1, 2)[page, at % T] = s["v"]
    return [_rotated(s, s["q"], at, s.get("q_weight")), s["k_pool"], s["v_pool"]]


def _rotated(s, x, positions, weight):
    """Heads [T, H, D], normed with weight and rotated by positions; angles in 64 bits, far positions lose them in 32."""
    R, half = s["case"]["rot"], s["case"]["layout"] == "half"
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight
    a = positions.double()[:, None] * s["angles"]
    cos, sin = (t.float().mul_(s["mscale"])[:, None] for t in (torch.cos(a), torch.sin(a)))
    r = y[..., :R]
    u, v = (r[..., :R // 2], r[..., R // 2:]) if half else (r[..., 0::2], r[..., 1::2])
    p, q = u * cos - v * sin, v * cos + u * sin
    r = torch.cat([p, q], -1) if half else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([r, y[..., R:]], -1).to(x.dtype)


def _grid(s):
    """(places [B, n] of the tokens of each sequence, clamped; whether there is one; sequence and place of every token)."""
    T = s["x"].shape[0]
    dev = s["x"].device
    if "cu" not in s:
        b = torch.arange(T, device=dev)
        return b[:, None], torch.ones(T, 1, dtype=torch.bool, device=dev), b, torch.zeros_like(b)
    cu, token = s["cu"].long(), torch.arange(T, device=dev)
    at = cu[:-1, None] + torch.arange(s["max_len"], device=dev)
    b = torch.searchsorted(cu[1:], token, right=True)
    return at.clamp(max=T - 1), at < cu[1:, None], b, token - cu[b]


def _conv_plain(s):
    x, state, rows = s["x"], s["conv"][0], s["rows"].long()
    W = s["weight"].shape[1]
    at, there, b, t = _grid(s)
    before = state[rows].float()
    if "held" in s:
        before = before * (s["held"] > 0)[:, None, None]
    padded = torch.cat([before, x[at].float()], 1)  # [B, W - 1 + n, C]
    n = at.shape[1]
    y = s["bias"] + sum(padded[:, j:j + n] * s["weight"][:, j] for j in range(W))
    y = F.silu(y)
    ends = there.sum(1)[:, None] + torch.arange(W - 1, device=x.device)
    state[rows] = padded[torch.arange(len(rows), device=x.device)[:, None], ends].to(x.dtype)
    return [y[b, t].to(x.dtype), s["conv"]]


def _steps(s, at, there):
    """Steps [B, n, H] in 64 bits: softplus(dt + bias), 0 where there is no token."""
    return F.softplus(s["dt"][at].double() + s["dt_bias"].double(), threshold=50.0) * there[:, :, None]


def _finish(s, y, x):
    """y + D x, gated: [T, H, P] of fp32 y."""
    y = y + s["D"][:, None] * x.float()
    return (y if s["z"] is None else y * F.silu(s["z"].float())).to(x.dtype)


def _step_plain(s):
    x, state, rows = s["x"], s["ssm"][0], s["rows"].long()
    G = s["case"]["heads"] // s["case"]["groups"]
    at, there, b, t = _grid(s)
    dt = _steps(s, at, there)[:, 0]
    dx = (x.double() * dt[:, :, None]).float()
    Bs, Cs = (s[n].float().repeat_interleave(G, 1) for n in ("B", "C"))
    h = state[rows] * torch.exp(dt * s["A"].double()).float()[:, :, None, None]
    h += dx[..., None] * Bs[:, :, None, :]
    state[rows] = h
    y = torch.matmul(h, Cs[..., None])[..., 0]
    return [_finish(s, y, x), s["ssm"]]


def _scan_plain(s):
    """In blocks of CHUNK tokens: products inside a block, the blocks' states joined by one product with their decays."""
    x, state, rows, L = s["x"], s["ssm"][0], s["rows"].long(), CHUNK
    T, H, P = x.shape
    G, N = s["B"].shape[1:]
    R = H // G
    at, there, b, t = _grid(s)
    nb = -(-at.shape[1] // L)
    at = F.pad(at, (0, nb * L - at.shape[1]))
    there = F.pad(there, (0, nb * L - there.shape[1]))
    B = len(rows)
    dt = _steps(s, at, there)  # [B, n, H], 64 bits
    sums = torch.cumsum((dt * s["A"].double()).view(B, nb, L, H), 2).permute(0, 1, 3, 2).contiguous()  # [B, nb, H, L]
    dtf = dt.float().view(B, nb, L, H).permute(0, 1, 3, 2).contiguous()
    xs = x[at].view(B, nb, L, H, P).permute(0, 1, 3, 2, 4).float().contiguous()
    Bs, Cs = (s[k][at].view(B, nb, L, G, N).permute(0, 1, 3, 2, 4).float() for k in ("B", "C"))
    past = torch.tril(torch.ones(L, L, dtype=torch.bool, device=x.device))
    decay = torch.exp((sums[..., :, None] - sums[..., None, :]).masked_fill_(~past, -math.inf).float())
    inner = (torch.matmul(Cs, Bs.transpose(3, 4))[:, :, :, None] * decay.view(B, nb, G, R, L, L)).view(B, nb, H, L, L)
    y = torch.matmul(inner * dtf[..., None, :], xs)
    del inner, decay
    # What each block adds to the state, and what enters each block.
    last = sums[..., -1]
    weighed = xs * (torch.exp(last[..., None] - sums).float() * dtf)[..., None]
    adds = torch.matmul(weighed.reshape(B, nb, G, R, L, P).transpose(4, 5), Bs[:, :, :, None]).reshape(B, nb, H, P * N)
    held = state[rows]
    if "held" in s:
        held = held * (s["held"] > 0)[:, None, None, None]
    adds = torch.cat([held.view(B, 1, H, P * N), adds], 1).permute(0, 2, 1, 3)  # [B, H, 1 + nb, P N]
    total = F.pad(torch.cumsum(last, 1).permute(0, 2, 1), (1, 0))  # [B, H, 1 + nb]
    reach = torch.tril(torch.ones(nb + 1, nb + 1, dtype=torch.bool, device=x.device))
    reach = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill_(~reach, -math.inf)).float()
    states = torch.matmul(reach, adds).view(B, H, nb + 1, P, N)
    del adds
    state[rows] = states[:, :, nb]
    entering = states[:, :, :nb].permute(0, 2, 1, 3, 4).reshape(B, nb, G, R, P, N)
    off = torch.matmul(Cs[:, :, :, None], entering.transpose(4, 5)).reshape(B, nb, H, L, P)
    y += off * torch.exp(sums).float()[..., None]
    y = y.permute(0, 1, 3, 2, 4).reshape(B, nb * L, H, P)[b, t]
    return [_finish(s, y, x), s["ssm"]]


# ---------------------------------------------------------------- the least a pass has to do
def work(case):
    k, e = case["kind"], 2
    if k in ("conv", "scan"):
        lens = _seq_lens(case)
        T, n = sum(lens), len(lens)
    if k == "conv":
        C = case["channels"]
        return {"bytes": 2 * T * C * e + 2 * n * (WIDTH - 1) * C * e + C * (WIDTH + 1) * 4, "flops": 2 * WIDTH * T * C}
    if k == "scan":
        H, G, P, N = case["heads"], case["groups"], case["dim"], case["state"]
        kept = (1 if case["fresh"] and n == 1 else 2) * n * H * P * N * 4
        return {"bytes": T * (2 * H * P + 2 * G * N + (H * P if case["gate"] else 0) + H) * e + kept, "flops": 4 * T * H * P * N}
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    T = case["tokens"] * (case["batch"] if k == "append" else 1)
    heads = H + (2 * Hkv if k == "append" else Hkv)
    return {"bytes": 2 * T * heads * D * e, "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k == "conv":
        return _conv_exact(s)
    if k == "scan":
        return _scan_exact(s)
    if k == "rotate":
        return tuple(_rotate_exact(s, s[n], s["positions"], s.get(n + "_weight")) for n in ("q", "k"))
    page, m = case["page"], case["tokens"]
    table, lens = s["table"].cpu().numpy(), s["lens"].tolist()
    at = np.concatenate([np.arange(n - m, n) for n in lens])
    pos = torch.from_numpy(at).cuda()
    pools = [s["k_pool"].double(), s["v_pool"].double()]
    for new, pool in zip((_rotate_exact(s, s["k"], pos, s.get("k_weight")), s["v"].double()), pools):
        for i, p in enumerate(at.tolist()):
            pool[0, int(table[i // m, p // page]), :, p % page] = new[i]
    return [_rotate_exact(s, s["q"], pos, s.get("q_weight"))] + pools


def _rotate_exact(s, x, positions, weight):
    """Each pair as a complex number times exp(i a)."""
    y, R = x.double(), s["case"]["rot"]
    if weight is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    half = s["case"]["layout"] == "half"
    i = torch.arange(R // 2, device=x.device)
    first, second = (i, i + R // 2) if half else (2 * i, 2 * i + 1)
    turn = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device=x.device), positions.double()[:, None] * s["angles"])
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _spans(s):
    if "cu" not in s:
        return [(i, i + 1) for i in range(s["x"].shape[0])]
    cu = s["cu"].tolist()
    return list(zip(cu, cu[1:]))


def _conv_exact(s):
    x, w, state = s["x"].double(), s["weight"].double(), s["conv"].double()
    out = torch.empty_like(x)
    held = s["held"].tolist() if "held" in s else None
    for i, ((a, b), row) in enumerate(zip(_spans(s), s["rows"].tolist())):
        seen = [state[0, row] if held is None or held[i] else torch.zeros_like(state[0, row]), x[a:b]]
        seen = torch.cat(seen)
        y = s["bias"].double().repeat(b - a, 1)
        for j in range(WIDTH):
            y += seen[j:j + b - a] * w[:, j]
        out[a:b] = y / (1 + torch.exp(-y))
        state[0, row] = seen[-(WIDTH - 1):]
    return [out, state]


def _scan_exact(s):
    """Token after token, all sequences side by side."""
    x, A = s["x"].double(), s["A"].double()
    T, H, P = x.shape
    R = H // s["B"].shape[1]
    raw = s["dt"].double() + s["dt_bias"].double()
    dt = torch.where(raw > 40, raw, torch.log1p(torch.exp(raw.clamp(max=40))))
    grow, dx = torch.exp(dt * A), x * dt[..., None]
    state, spans, rows = s["ssm"].double(), _spans(s), s["rows"].long()
    h = state[0, rows]
    if "held" in s:
        h[s["held"] == 0] = 0
    y = torch.empty_like(x)
    order = sorted(range(len(spans)), key=lambda i: spans[i][0] - spans[i][1])  # the longest first: those that are left are the first ones
    h = h[order]
    starts = np.array([spans[i][0] for i in order])
    lens = np.array([spans[i][1] - spans[i][0] for i in order])
    on_device = torch.from_numpy(starts).cuda()
    for t in range(int(lens[0])):
        n = int((lens > t).sum())
        at = on_device[:n] + t
        Bt, Ct = (s[k][at].double().repeat_interleave(R, 1) for k in ("B", "C"))
        h[:n] = h[:n] * grow[at][..., None, None] + dx[at][..., None] * Bt[:, :, None]
        y[at] = (h[:n] * Ct[:, :, None]).sum(-1)
    state[0, rows[torch.tensor(order, device=rows.device)]] = h
    y = y + s["D"].double()[:, None] * x
    if s["z"] is not None:
        z = s["z"].double()
        y = y * z / (1 + torch.exp(-z))
    return [y, state]
