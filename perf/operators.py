"""Performance cases of attention and its paged key/value cache, through the package's public calls.

Families (`kind`), each over the sizes a serving engine meets:
  prompt  causal attention over packed prompts of different lengths with grouped heads, attn.prompt;
          q is a column view of a wider projection (the gate lies beside it), as the decoder's is;
  paged   new tokens of each sequence over its cached ones, attn.paged: decode steps (one token a
          sequence) and prompt chunks;
  shared  one token of each sequence of a batch whose sequences share a long prefix,
          attn.shared_prefix;
  append  a step's keys and values into one layer's pages, KVCache.append;
  fork    sequences freed and forked again (a search's beams, parallel samples), KVCache.free and
          KVCache.fork: full pages shared, part-filled ones copied in every layer;
  compact the live pages moved to the front of a fragmented pool, KVCache.compact, into tables of
          their own.

q and k are N(0, 1) as behind a norm, v is N(0, 1); pages lie in the pool in random order. Lengths of a
batch are spread over the logarithm of their range, the same for every seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # Three short prompts that arrive together, one of a single token: the shortest prefill.
        dict(name="prompt_f16_short", kind="prompt", dtype="f16", lens="1,7,19", heads=48, kv_heads=8, dim=128),
        # An ordinary ragged batch of prompts, the lengths a scheduler packs into one step.
        dict(name="prompt_bf16_ragged", kind="prompt", dtype="bf16", lens="1008,333,64,1,511,129", heads=48,
             kv_heads=8, dim=128),
        # Two longer prompts on heads of 256 (the decoder's 6144 | 1024 wide q and k).
        dict(name="prompt_f16_d256", kind="prompt", dtype="f16", lens="2048,1531", heads=24, kv_heads=4, dim=256),
        # One long prompt: the largest prefill.
        dict(name="prompt_bf16_8192", kind="prompt", dtype="bf16", lens="8192", heads=48, kv_heads=8, dim=128),
        # A split-fuse step's 64-token prompt chunk on top of 6000 cached tokens.
        dict(name="chunk_bf16_64_on_6000", kind="paged", dtype="bf16", batch=1, tokens=64, lo=6064, hi=6064, heads=48,
             kv_heads=8, dim=128, page=64),
        # One chat, one token, a short history: the decode step where latency counts.
        dict(name="decode_f16_1", kind="paged", dtype="f16", batch=1, tokens=1, lo=777, hi=777, heads=48, kv_heads=8,
             dim=128, page=16),
        # A full decode batch of ragged histories on heads of 256.
        dict(name="decode_bf16_16", kind="paged", dtype="bf16", batch=16, tokens=1, lo=37, hi=8192, heads=24,
             kv_heads=4, dim=256, page=64),
        # 64 sessions under one system prompt, each with its own turns behind it.
        dict(name="shared_f16_64", kind="shared", dtype="f16", batch=64, groups=1, prefix=4011, lo=1, hi=512, heads=48,
             kv_heads=8, dim=128, page=64),
        # 128 sessions over two long documents: the largest decode step.
        dict(name="shared_bf16_128", kind="shared", dtype="bf16", batch=128, groups=2, prefix=32768, lo=16, hi=1024,
             heads=48, kv_heads=8, dim=128, page=64),
        # A split-fuse step's 80 new tokens into one layer's pages.
        dict(name="append_bf16_80", kind="append", dtype="bf16", batch=80, tokens=1, lo=80, hi=4096, kv_heads=8, dim=128,
             page=64),
        # Eight sequences forked into four continuations each, in the 16 attention layers of the decoder.
        dict(name="fork_f16_32", kind="fork", dtype="f16", batch=8, children=4, lo=100, hi=2000, layers=16, kv_heads=4,
             dim=256, page=64),
        # A pool half of whose sequences have ended, compacted.
        dict(name="compact_bf16_512", kind="compact", dtype="bf16", pages=512, live=0.5, layers=16, kv_heads=4,
             dim=256, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _heads(rng):
    """Grouped heads: the decoder's widths, and other common ratios."""
    return rng.choice([(48, 8, 128), (24, 4, 256), (32, 8, 128), (16, 16, 64), (32, 4, 64), (40, 8, 128), (8, 1, 128),
                       (16, 2, 256)])


def _draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "paged", "paged", "paged", "shared", "shared", "shared", "append",
                       "fork", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    H, Hkv, D = _heads(rng)
    page = rng.choice([16, 32, 64, 128])
    if kind == "prompt":
        n = rng.randint(1, 8)
        top = _log_int(rng, 16, 8192)
        return dict(kind=kind, dtype=dtype, lens=",".join(str(_log_int(rng, 1, top)) for _ in range(n)), heads=H,
                    kv_heads=Hkv, dim=D)
    if kind == "paged":
        hi = _log_int(rng, 64, 16384)
        tokens = rng.choice([1, 1, 1, 4, 64, _log_int(rng, 1, 512)])
        hi = max(hi, tokens)
        lo = max(tokens, _log_int(rng, 1, hi))
        return dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 64 if tokens < 16 else 4), tokens=tokens, lo=lo, hi=hi,
                    heads=H, kv_heads=Hkv, dim=D, page=page)
    if kind == "shared":
        hi = _log_int(rng, 8, 1024)
        batch = _log_int(rng, 2, 128)
        return dict(kind=kind, dtype=dtype, batch=batch, groups=min(batch, rng.choice([1, 1, 2, 5])),
                    prefix=_log_int(rng, 64, 32768), lo=_log_int(rng, 1, hi), hi=hi, heads=H, kv_heads=Hkv, dim=D, page=page)
    if kind == "append":
        tokens = rng.choice([1, 1, 64, _log_int(rng, 1, 512)])
        hi = max(tokens, _log_int(rng, 64, 8192))
        return dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 128 if tokens == 1 else 8), tokens=tokens,
                    lo=max(tokens, _log_int(rng, 1, hi)), hi=hi, kv_heads=Hkv, dim=D, page=page)
    if kind == "fork":
        hi = _log_int(rng, 32, 4096)
        return dict(kind=kind, dtype=dtype, batch=rng.randint(1, 16), children=rng.randint(1, 8), lo=_log_int(rng, 1, hi),
                    hi=hi, layers=rng.choice([4, 16]), kv_heads=Hkv, dim=D, page=page)
    return dict(kind=kind, dtype=dtype, pages=_log_int(rng, 64, 512), live=round(rng.uniform(0.2, 0.8), 3),
                layers=rng.choice([4, 16]), kv_heads=Hkv, dim=D, page=page)


def _cost(case):
    """What the plain form of a case costs, by the bytes of its scores or of its pool."""
    k = case["kind"]
    if k == "prompt":
        n = [int(x) for x in case["lens"].split(",")]
        return len(n) * max(n) ** 2 * case["heads"] * 4
    if k == "paged":
        return case["batch"] * case["hi"] * (case["tokens"] * case["heads"] + 4 * case["heads"] * case["dim"]) * 4
    if k == "shared":
        return case["batch"] * case["heads"] * (case["prefix"] + case["hi"] * 4 * case["dim"]) * 4
    return 2 * _pool_pages(case) * case.get("layers", 1) * case["page"] * case["kv_heads"] * case["dim"] * 2


def _load(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 8e14


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, ragged ones among them; none with more
    work, or a larger plain form, than the listed ones."""
    kinds = {"prompt": ("prompt",), "paged": ("paged", "shared"), "shared": ("paged", "shared"), "append": ("append", "fork", "compact"),
             "fork": ("fork", "compact"), "compact": ("fork", "compact")}
    while True:
        c = _draw(rng)
        peers = [x for x in listed() if x["kind"] in kinds[c["kind"]]]
        if _load(c) <= max(_load(x) for x in peers) and _cost(c) <= max(_cost(x) for x in peers):
            return c


# ---------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n lengths over the logarithm of lo..hi, both ends among them, in a scattered order."""
    u = [(i * 0.6180339887498949) % 1.0 for i in range(n)]
    got = [int(round(lo * (hi / lo) ** x)) for x in u]
    got[-1] = hi
    return [min(max(x, lo), hi) for x in got]


def _lens(case):
    """The cached tokens of each sequence, new ones included (a shared prefix too)."""
    return [case.get("prefix", 0) + x for x in _spread(case["batch"], case["lo"], case["hi"])]


def _group_starts(case):
    B, n = case["batch"], case["groups"]
    return [B * i // n for i in range(n)] + [B]


def _pool_pages(case):
    """Pages of the pool: what the sequences hold, and an eighth more."""
    k, T = case["kind"], case["page"]
    if k == "compact":
        return case["pages"]
    if k == "shared":
        P = case["prefix"]
        return _grown(case["groups"] * (P // T) + sum(-(-n // T) - P // T for n in _lens(case)))
    if k == "fork":
        return _grown(sum(-(-n // T) + case["children"] for n in _lens(case)))
    return _grown(sum(-(-n // T) for n in _lens(case)))


def _grown(n):
    return n + n // 8 + 1


def _randn(gen, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)


def _tables(case, rng):
    """(table, lens, refs) of a cache whose pages were taken from a pool in random order."""
    k, T, P = case["kind"], case["page"], _pool_pages(case)
    order = rng.permutation(P)
    if k == "compact":
        # Sequences of 1 to 8 pages fill the pool, then all but a share of them end.
        sizes, left, spread = [], P, np.random.default_rng(1)  # the same sizes for every seed
        while left:
            n = min(left, int(spread.integers(1, 9)))
            sizes.append(n)
            left -= n
        keep = rng.permutation(len(sizes))[:max(1, int(round(case["live"] * len(sizes))))]
        lens = np.zeros(len(sizes), np.int64)
        table = np.full((len(sizes), 8), -1, np.int64)
        at = np.concatenate([[0], np.cumsum(sizes)])
        for i in keep:
            table[i, :sizes[i]] = order[at[i]:at[i + 1]]
            lens[i] = sizes[i] * T - int(rng.integers(0, T))
    else:
        lens = np.array(_lens(case))
        used = -(-lens // T)
        rows = len(lens) * (1 + case.get("children", 0))
        table = np.full((rows, int(used.max()) + 1), -1, np.int64)
        at = 0
        if k == "shared":
            full, g = case["prefix"] // T, _group_starts(case)
            for a, b in zip(g, g[1:]):
                table[a:b, :full] = order[at:at + full]
                at += full
        else:
            full = 0
        for i, n in enumerate(used):
            table[i, full:n] = order[at:at + n - full]
            at += n - full
        lens = np.concatenate([lens, np.zeros(rows - len(lens), np.int64)])
    refs = np.bincount(table[table >= 0], minlength=P)
    return table, lens, refs


def _fork_ints(table, lens, refs, parents, children, T):
    """The bookkeeping after every child has been forked from its parent: also (source, copy, tokens) of the
    part-filled pages."""
    table, lens, refs = table.copy(), lens.copy(), refs.copy()
    moves = []
    for p, c in zip(parents, children):
        full, part = divmod(int(lens[p]), T)
        table[c] = -1
        table[c, :full] = table[p, :full]
        refs[table[p, :full]] += 1
        if part:
            new = int(np.flatnonzero(refs == 0)[0])
            moves.append((int(table[p, full]), new, part))
            table[c, full] = new
            refs[new] = 1
        lens[c] = lens[p]
    return table, lens, refs, moves


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    k, dt = case["kind"], DTYPES[case["dtype"]]
    D, Hkv, H = case["dim"], case["kv_heads"], case.get("heads", 0)
    s = {"case": case, "scale": 1.0 / math.sqrt(D)}
    if k == "prompt":
        lens = [int(x) for x in case["lens"].split(",")]
        T = sum(lens)
        s["cu"] = _i32(np.concatenate([[0], np.cumsum(lens)]))
        s["max_q"] = max(lens)
        # The projections' outputs: q with its gate beside it, k and v.
        s["q"] = _randn(gen, dt, T, 2 * H * D)[:, :H * D].view(T, H, D)
        s["k"] = _randn(gen, dt, T, Hkv * D).view(T, Hkv, D)
        s["v"] = _randn(gen, dt, T, Hkv * D).view(T, Hkv, D)
        return s
    P, T, L = _pool_pages(case), case["page"], case.get("layers", 1)
    table, lens, refs = _tables(case, rng)
    pool_k, pool_v = _randn(gen, dt, L, P, Hkv, T, D), _randn(gen, dt, L, P, Hkv, T, D)
    if k == "fork":
        n = case["batch"]
        s["parents"] = np.repeat(np.arange(n), case["children"])
        s["children"] = np.arange(n * case["children"]) + n
        table, lens, refs, _ = _fork_ints(table, lens, refs, s["parents"], s["children"], T)
        s["parents"], s["children"] = _i32(s["parents"]), _i32(s["children"])
    s.update(k=pool_k, v=pool_v, table=_i32(table), lens=_i32(lens), refs=_i32(refs))
    if k == "compact":
        s["new_table"], s["new_refs"] = torch.empty_like(s["table"]), torch.empty_like(s["refs"])
    else:
        s["rows"] = torch.arange(case["batch"], dtype=torch.int32, device="cuda")
        s["max_len"] = int(lens.max())
    if k in ("paged", "append") and case["tokens"] > 1:
        s["cu"] = torch.arange(case["batch"] + 1, dtype=torch.int32, device="cuda") * case["tokens"]
    if k == "paged":
        N = case["batch"] * case["tokens"]
        s["q"] = _randn(gen, dt, N, 2 * H * D)[:, :H * D].view(N, H, D)
    if k == "shared":
        s["q"] = _randn(gen, dt, case["batch"], 2 * H * D)[:, :H * D].view(case["batch"], H, D)
        s["starts"] = _i32(_group_starts(case))
        s["prefix"] = torch.full((case["groups"],), case["prefix"], dtype=torch.int32, device="cuda")
    if k == "append":
        N = case["batch"] * case["tokens"]
        s["k_new"], s["v_new"] = _randn(gen, dt, N, Hkv, D), _randn(gen, dt, N, Hkv, D)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)(s, s["case"]["kind"])


def _run_own(s, k):
    from nebula_amd import attn

    if k == "prompt":
        return attn.prompt(s["q"], s["k"], s["v"], s["cu"], scale=s["scale"], with_lse=True)
    if "cache" not in s:  # the handle that a program makes once
        s["cache"] = attn.KVCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    c = s["cache"]
    if k == "paged":
        return attn.paged(s["q"], c, 0, s["rows"], cu_seqlens=s.get("cu"), max_len=s["max_len"], scale=s["scale"])
    if k == "shared":
        return attn.shared_prefix(s["q"], c, 0, s["rows"], s["starts"], s["prefix"], max_prefix=s["case"]["prefix"],
                                  max_len=s["max_len"], scale=s["scale"])
    if k == "append":
        c.append(0, s["k_new"], s["v_new"], s["rows"], cu_seqlens=s.get("cu"))
        return [s["k"], s["v"]]
    if k == "fork":
        c.free(s["children"])
        c.fork(s["parents"], s["children"])
        return [s["k"], s["v"], s["table"], s["lens"], s["refs"]]
    c.compact(out_table=s["new_table"], out_refs=s["new_refs"])
    return [s["k"], s["v"], s["new_table"], s["new_refs"]]


def _softmax_pv(scores, allowed, v):
    """Softmax over the last axis where allowed, times v; and the logarithm of its sum. Rows with no key give 0."""
    m = scores.masked_fill(~allowed, -math.inf).amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = torch.exp(scores.sub_(m)).masked_fill_(~allowed, 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(l > 0, l, torch.ones_like(l))
    return o, (m + torch.log(l)).squeeze(-1)


def _pad(x, starts, n):
    """Rows [starts[b], starts[b] + n) of x, clamped to the last, as [B, n, ...]."""
    at = starts[:, None].long() + torch.arange(n, device=x.device)
    return x[at.clamp_(max=x.shape[0] - 1)].float()


def _gathered(pool, table, n):
    """The first n tokens of each sequence of one layer's pool [P, Hkv, T, D]: [B, Hkv, n, D]."""
    T = pool.shape[2]
    j = torch.arange(n, device=pool.device)
    page = table[:, j // T].long().clamp(min=0)
    return pool.transpose(1, 2)[page, j % T].permute(0, 2, 1, 3).float()


def _run_plain(s, k):
    case = s["case"]
    if k == "prompt":
        q, cu, n = s["q"], s["cu"], s["max_q"]
        T, H, D = q.shape
        Hkv, B = s["k"].shape[1], cu.shape[0] - 1
        lens = (cu[1:] - cu[:-1]).long()
        qs = _pad(q, cu[:-1], n).view(B, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, H // Hkv * n, D)
        ks = _pad(s["k"], cu[:-1], n).permute(0, 2, 3, 1)
        vs = _pad(s["v"], cu[:-1], n).permute(0, 2, 1, 3)
        scores = torch.matmul(qs, ks).mul_(s["scale"]).view(B, Hkv, H // Hkv, n, n)
        at = torch.arange(n, device=q.device)
        allowed = (at[None, :] <= at[:, None]) & (at[None, None, :] < lens[:, None, None])
        o, lse = _softmax_pv(scores, allowed[:, None, None], vs[:, :, None])
        token = torch.arange(T, device=q.device)
        b = torch.searchsorted(cu.long()[1:], token, right=True)
        t = token - cu.long()[b]
        o = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[b, t]
        return o.to(q.dtype), lse.permute(0, 3, 1, 2).reshape(B, n, H)[b, t]
    pool_k, pool_v, T, lens = s["k"], s["v"], case["page"], s["lens"].long()
    if k == "paged":
        q = s["q"]
        N, H, D = q.shape
        Hkv, B, m = pool_k.shape[2], case["batch"], case["tokens"]
        G, n = H // Hkv, s["max_len"]
        ks, vs = _gathered(pool_k[0], s["table"], n), _gathered(pool_v[0], s["table"], n)
        qs = q.float().view(B, m, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * m, D)
        scores = torch.matmul(qs, ks.transpose(2, 3)).mul_(s["scale"]).view(B, Hkv, G, m, n)
        last = lens[:, None] - m + torch.arange(m, device=q.device)
        allowed = torch.arange(n, device=q.device) <= last[:, :, None]
        o, _ = _softmax_pv(scores, allowed[:, None, None], vs[:, :, None])
        return o.permute(0, 3, 1, 2, 4).reshape(N, H, D).to(q.dtype)
    if k == "shared":
        q, P = s["q"], case["prefix"]
        B, H, D = q.shape
        Hkv, full = pool_k.shape[2], P // T * T
        G, n = H // Hkv, s["max_len"] - full
        group = torch.searchsorted(s["starts"][1:].long(), torch.arange(B, device=q.device), right=True)
        # The prefix's whole pages once for each group, with every query of the batch against them; a query keeps its own.
        first = s["table"][s["starts"][:-1].long()]
        kp, vp = _gathered(pool_k[0], first, full), _gathered(pool_v[0], first, full)
        ks, vs = _gathered(pool_k[0], s["table"][:, full // T:], n), _gathered(pool_v[0], s["table"][:, full // T:], n)
        qs = q.float().view(B, Hkv, G, D)
        heads = qs.permute(1, 0, 2, 3).reshape(1, Hkv, B * G, D)
        sp = torch.matmul(heads, kp.transpose(2, 3)).mul_(s["scale"]).view(-1, Hkv, B, G, full)
        sp = sp[group, :, torch.arange(B, device=q.device)]
        ss = torch.matmul(qs, ks.transpose(2, 3)).mul_(s["scale"])
        ss = ss.masked_fill_(torch.arange(full, full + n, device=q.device) >= lens[:, None, None, None], -math.inf)
        m = torch.maximum(sp.amax(-1, keepdim=True) if full else ss.amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
        sp, ss = torch.exp(sp.sub_(m)), torch.exp(ss.sub_(m))
        l = sp.sum(-1, keepdim=True) + ss.sum(-1, keepdim=True)
        mine = torch.arange(kp.shape[0], device=q.device)[:, None] == group
        sp = (sp[None] * mine[:, :, None, None, None]).permute(0, 2, 1, 3, 4).reshape(-1, Hkv, B * G, full)
        o = torch.matmul(sp, vp).sum(0).view(Hkv, B, G, D).permute(1, 0, 2, 3) + torch.matmul(ss, vs)
        return (o / l).reshape(B, H, D).to(q.dtype)
    if k == "append":
        m = case["tokens"]
        at = (lens[:, None] - m + torch.arange(m, device=lens.device)).reshape(-1)
        row = torch.arange(case["batch"], device=lens.device).repeat_interleave(m)
        page = s["table"][row, at // T].long()
        pool_k[0].transpose(1, 2)[page, at % T] = s["k_new"]
        pool_v[0].transpose(1, 2)[page, at % T] = s["v_new"]
        return [pool_k, pool_v]
    if k == "fork":
        return _fork_plain(s, T)
    return _compact_plain(s)


def _fork_plain(s, T):
    table, lens, refs = s["table"], s["lens"], s["refs"]
    par, kid = s["parents"].long(), s["children"].long()
    gone = table[kid]
    refs -= torch.bincount(gone[gone >= 0], minlength=refs.numel()).int()
    n = lens[par].long()
    full, part = n // T, n % T
    col = torch.arange(table.shape[1], device=table.device)
    kids = torch.where(col < full[:, None], table[par], -1)
    refs += torch.bincount(kids[kids >= 0], minlength=refs.numel()).int()
    some = (part > 0).nonzero().squeeze(1)
    new = (refs == 0).nonzero().squeeze(1)[:some.numel()]
    src = table[par[some], full[some]].long()
    kids[some, full[some]] = new.int()
    refs[new] = 1
    table[kid] = kids
    lens[kid] = lens[par]
    keep = (torch.arange(T, device=table.device) < part[some][:, None])[None, :, None, :, None]
    s["k"][:, new] = torch.where(keep, s["k"][:, src], s["k"][:, new])
    s["v"][:, new] = torch.where(keep, s["v"][:, src], s["v"][:, new])
    return [s["k"], s["v"], table, lens, refs]


def _compact_plain(s):
    refs, table = s["refs"], s["table"]
    live = refs > 0
    at = torch.arange(refs.numel(), device=refs.device)
    n = live.sum()
    src, dst = (live & (at >= n)).nonzero().squeeze(1), (~live & (at < n)).nonzero().squeeze(1)
    to = at.clone()
    to[src] = dst
    s["new_table"].copy_(torch.where(table >= 0, to[table.long().clamp(min=0)], -1))
    s["new_refs"].copy_(refs)
    s["new_refs"][dst] = refs[src]
    s["new_refs"][src] = 0
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return [s["k"], s["v"], s["new_table"], s["new_refs"]]


# ---------------------------------------------------------------- the least a pass has to do
def work(case):
    k, D, Hkv, e = case["kind"], case["dim"], case["kv_heads"], 2
    H = case.get("heads", 0)
    if k == "prompt":
        lens = [int(x) for x in case["lens"].split(",")]
        T = sum(lens)
        return {"bytes": T * (2 * H * D * e + 2 * Hkv * D * e + 4 * H), "flops": 4 * D * H * sum(n * (n + 1) // 2 for n in lens)}
    token = 2 * Hkv * D * e  # a token's key and value in one layer
    if k == "paged":
        m, lens = case["tokens"], _lens(case)
        return {"bytes": sum(lens) * token + case["batch"] * m * 2 * H * D * e,
                "flops": 4 * D * H * sum(m * n - m * (m - 1) // 2 for n in lens)}
    if k == "shared":
        P, lens = case["prefix"], _lens(case)
        return {"bytes": (case["groups"] * P + sum(n - P for n in lens)) * token + case["batch"] * 2 * H * D * e,
                "flops": 4 * D * H * sum(lens)}
    if k == "append":
        return {"bytes": 2 * case["batch"] * case["tokens"] * token, "flops": 0}
    if k == "fork":
        T, lens = case["page"], _lens(case)
        pages = sum(-(-n // T) for n in lens) * case["children"]
        part = sum(n % T for n in lens) * case["children"]
        return {"bytes": 2 * part * case["layers"] * token + 16 * pages, "flops": 0}
    table, lens, refs = _tables(case, np.random.default_rng(0))
    live = int((refs > 0).sum())
    moved = int((refs[live:] > 0).sum())
    return {"bytes": 2 * moved * case["page"] * case["layers"] * token + 8 * (table.size + refs.size), "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_rows(q, k, v, limits, scale):
    """softmax(scale q k^T) v and the logarithm of its sum, row r over keys [0, limits[r]); one head, 64 bits."""
    s = (q.double() @ k.double().T) * scale
    s[torch.arange(k.shape[0], device=s.device)[None, :] >= limits[:, None]] = -math.inf
    lse = torch.logsumexp(s, 1)
    return torch.exp(s - lse[:, None]) @ v.double(), lse


def _tokens_of(pool, pages, n):
    """The first n tokens of a sequence, one kv head: pool [P, T, D]."""
    return pool[pages.long()].reshape(-1, pool.shape[-1])[:n]


def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k in ("prompt", "paged", "shared"):
        q = s["q"]
        N, H, D = q.shape
        G = H // case["kv_heads"]
        out = torch.empty(N, H, D, dtype=torch.float64, device=q.device)
        lse = torch.empty(N, H, dtype=torch.float64, device=q.device)
        if k == "prompt":
            ends = np.cumsum([int(x) for x in case["lens"].split(",")]).tolist()
            spans = list(zip([0] + ends[:-1], ends))
        else:
            m = case.get("tokens", 1)
            spans = [(i * m, i * m + m) for i in range(case["batch"])]
            table, lens = s["table"].cpu(), s["lens"].tolist()
        for i, (a, b) in enumerate(spans):
            n = b - a if k == "prompt" else lens[i]
            limits = torch.arange(n - (b - a), n, device=q.device) + 1
            for g in range(case["kv_heads"]):
                if k == "prompt":
                    kk, vv = s["k"][a:b, g], s["v"][a:b, g]
                else:
                    pages = table[i, :-(-n // case["page"])].to(q.device)
                    kk, vv = _tokens_of(s["k"][0][:, g], pages, n), _tokens_of(s["v"][0][:, g], pages, n)
                for h in range(g * G, g * G + G) if k == "prompt" else [slice(g * G, g * G + G)]:
                    rows = q[a:b, h].reshape(-1, D)
                    o, e = _exact_rows(rows, kk, vv, limits if k == "prompt" else limits.repeat_interleave(G), s["scale"])
                    out[a:b, h], lse[a:b, h] = o.view(out[a:b, h].shape), e.view(lse[a:b, h].shape)
        return (out, lse) if k == "prompt" else out
    T = case["page"]
    table, lens, refs = (s[x].cpu().numpy().astype(np.int64) for x in ("table", "lens", "refs"))
    pools = [s["k"], s["v"]]
    if k == "append":
        m = case["tokens"]
        for new, pool in ((s["k_new"], s["k"]), (s["v_new"], s["v"])):
            for i in range(case["batch"]):
                for t in range(m):
                    at = int(lens[i]) - m + t
                    pool[0, int(table[i, at // T]), :, at % T] = new[i * m + t]
        return [p.double() for p in pools]
    if k == "fork":
        par, kid = s["parents"].tolist(), s["children"].tolist()
        for c in kid:
            np.subtract.at(refs, table[c][table[c] >= 0], 1)
        table, lens, refs, moves = _fork_ints(table, lens, refs, par, kid, T)
        for src, dst, part in moves:
            for p in pools:
                p[:, dst, :, :part] = p[:, src, :, :part].clone()
        return [p.double() for p in pools] + [_i32(table), _i32(lens), _i32(refs)]
    live = np.flatnonzero(refs)
    holes = np.flatnonzero(refs[:len(live)] == 0)
    movers = live[live >= len(live)]
    to = np.arange(len(refs))
    new_refs = refs.copy()
    for src, dst in zip(movers.tolist(), holes.tolist()):
        to[src] = dst
        new_refs[dst], new_refs[src] = refs[src], 0
        for p in pools:
            p[:, dst] = p[:, src].clone()
    return [p.double() for p in pools] + [_i32(np.where(table >= 0, to[np.maximum(table, 0)], -1)), _i32(new_refs)]
