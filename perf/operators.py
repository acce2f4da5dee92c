"""Measured cases of the operators that serve many takes from one prompt.

Three families: attention for a batch that shares a long prefix (``prefix_attn``), the pages
of the cache it reads (``pages_fork`` / ``pages_free`` / ``pages_compact`` / ``pages_grow`` and
the paged RoPE/KV write ``rope_pages``), and the matrix product in 8-bit integers with a scale
for each token and each output channel (``int8_mm_a8``).

``run`` computes an operator in its plain form (elementary torch operations, 32 bits, rounded
once at the end), or, with ``own``, through the framework's entry points.  ``exact`` gives the
same outputs from the definitions in 64 bits.

Cache layout: ``k``, ``v`` ``[layers, pages, Hk, page, hd]`` (one layer of it for the attention
and the write); ``table [sequences, pages of a sequence]`` int32, -1 where a sequence holds no
page; ``lens [sequences]`` int64 positions held; ``refs [pages]`` int32 sequences that hold a
page, 0 = free.  Free pages are handed out lowest number first, in the order of the call's list.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the first frame after a prompt, one take: only latency counts
        dict(name="attn-first-frame", op="attn", B=1, groups=1, S=1, Hq=24, Hk=8, hd=128, page=64, prefix=512,
             own_max=1, ragged=False, pad=False, dtype="fp16"),
        # four takes and their unconditional rows in the middle of a song, two prompts
        dict(name="attn-takes", op="attn", B=8, groups=2, S=1, Hq=24, Hk=8, hd=128, page=64, prefix=600,
             own_max=750, ragged=True, pad=False, dtype="fp16"),
        # a server's batch on one system prompt, short answers so far, small pages
        dict(name="attn-crowd", op="attn", B=64, groups=1, S=1, Hq=32, Hk=8, hd=128, page=32, prefix=4096,
             own_max=512, ragged=True, pad=True, dtype="bf16"),
        # two long documents with eight questions each
        dict(name="attn-long", op="attn", B=16, groups=2, S=1, Hq=24, Hk=8, hd=128, page=64, prefix=30001,
             own_max=2000, ragged=True, pad=False, dtype="fp16"),
        # one hypothesis forked in a small decoder
        dict(name="fork-one", op="fork", layers=4, n_src=1, n_dst=1, n_pages=24, Hk=2, hd=128, page=16, length=37,
             dtype="fp16"),
        # a conditional and an unconditional prompt forked into four takes each
        dict(name="fork-takes", op="fork", layers=28, n_src=2, n_dst=8, n_pages=40, Hk=8, hd=128, page=64, length=600,
             dtype="fp16"),
        # a pool with every other page free is packed before it is handed back
        dict(name="compact-pool", op="compact", layers=16, n_pages=128, n_seqs=12, live=0.5, Hk=8, hd=128, page=64,
             dtype="fp16"),
        # a chunk of two prompts enters the cache: pages taken, RoPE, K and V written
        dict(name="write-prompt", op="write", B=2, S=500, start=300, Hq=24, Hk=8, hd=128, page=64, dtype="fp16"),
        # one token through a projection
        dict(name="mm-token", op="mm", M=1, N=5120, K=4096, silu=False, res=False, dtype="fp16"),
        # eight rows of a frame through a gated MLP's first half
        dict(name="mm-takes", op="mm", M=8, N=16384, K=4096, silu=True, res=False, dtype="fp16"),
        # a short prompt of odd length, added to the residual stream
        dict(name="mm-short-prompt", op="mm", M=333, N=4096, K=2048, silu=False, res=True, dtype="bf16"),
        # a batch of prompts through the gated MLP's first half
        dict(name="mm-prompts", op="mm", M=4096, N=16384, K=4096, silu=True, res=False, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _draw_attn(rng):
    B = _log(rng, 1, 64)
    S = rng.choice([1, 1, 1, 2, 3, 8])
    Hk = rng.choice([1, 2, 4, 8])
    return dict(op="attn", B=B, groups=rng.randint(1, min(B, 4)), S=S, Hq=Hk * rng.choice([1, 2, 3, 4, 7, 8]), Hk=Hk,
                hd=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]), prefix=_log(rng, 1, 30000),
                own_max=max(S, _log(rng, 1, 2000)), ragged=rng.random() < 0.8, pad=rng.random() < 0.3,
                dtype=rng.choice(["fp16", "bf16"]))


def _draw_fork(rng):
    n_src, page, length = _log(rng, 1, 8), rng.choice([16, 32, 64, 128]), _log(rng, 1, 1500)
    n_dst = _log(rng, 1, 32)
    return dict(op="fork", layers=_log(rng, 1, 28), n_src=n_src, n_dst=n_dst,
                n_pages=n_src * -(-length // page) + n_dst + rng.randint(0, 8), Hk=rng.choice([1, 2, 4, 8]),
                hd=rng.choice([64, 128, 256]), page=page, length=length, dtype=rng.choice(["fp16", "bf16"]))


def _draw_compact(rng):
    n_pages = _log(rng, 8, 1500)
    return dict(op="compact", layers=_log(rng, 1, 28), n_pages=n_pages, n_seqs=_log(rng, 1, min(64, n_pages // 4)),
                live=rng.uniform(0.2, 0.9), Hk=rng.choice([1, 2, 4, 8]), hd=rng.choice([64, 128, 256]),
                page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]))


def _draw_write(rng):
    S = _log(rng, 1, 1000)
    Hk = rng.choice([1, 2, 4, 8])
    return dict(op="write", B=_log(rng, 1, 64 if S < 16 else 4), S=S, start=rng.randint(0, 2000),
                Hq=Hk * rng.choice([1, 2, 3, 4, 8]), Hk=Hk, hd=rng.choice([64, 128, 256]),
                page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]))


def _draw_mm(rng):
    silu = rng.random() < 0.4
    N = 32 * _log(rng, 4, 512) if silu or rng.random() < 0.7 else _log(rng, 100, 16384)
    return dict(op="mm", M=_log(rng, 1, 4096), N=N, K=16 * _log(rng, 4, 512), silu=silu,
                res=not silu and rng.random() < 0.5, dtype=rng.choice(["fp16", "bf16"]))


def _cost(case):
    """(bytes moved, flops, bytes of the pool) that bound what a drawn case may cost."""
    w = work(case)
    pool = 0
    if case["op"] in ("fork", "compact"):
        pool = 4 * case["layers"] * case["n_pages"] * case["Hk"] * case["page"] * case["hd"]
    if case["op"] == "attn":   # the plain form gathers every sequence's whole history in 32 bits
        pool = 4 * case["B"] * (case["prefix"] + case["own_max"]) * case["Hk"] * case["hd"]
    return w["bytes"], w["flops"], pool


def draw(rng):
    kind = rng.choice(["attn", "attn", "pages", "mm", "mm"])
    while True:
        if kind == "pages":
            case = rng.choice([_draw_fork, _draw_compact, _draw_write])(rng)
        else:
            case = {"attn": _draw_attn, "mm": _draw_mm}[kind](rng)
        top = [_cost(c) for c in listed() if c["op"] == case["op"]]
        if all(x <= max(t[i] for t in top) for i, x in enumerate(_cost(case))):
            return case


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _ints(case, seed, n, lo, hi):
    """n whole numbers in [lo, hi] on the host (lengths, orders)."""
    g = torch.Generator()
    g.manual_seed(seed * 7919 + 17)
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _perm(seed, n):
    g = torch.Generator()
    g.manual_seed(seed * 104729 + 5)
    return torch.randperm(n, generator=g).tolist()


def _attn_lens(case, seed):
    """Positions that each sequence holds beyond the prefix; -1: a padding row."""
    B, S = case["B"], case["S"]
    lens = _ints(case, seed, B, S, case["own_max"]) if case["ragged"] else [case["own_max"]] * B
    if case["pad"] and B > 1:
        lens[B // 2] = -1
    return lens


def _gstart(case):
    B, n = case["B"], case["groups"]
    return [B * i // n for i in range(n + 1)]


def _prep_attn(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    B, S, Hq, Hk, hd, page, P = (case[x] for x in ("B", "S", "Hq", "Hk", "hd", "page", "prefix"))
    lens, gs = _attn_lens(case, seed), _gstart(case)
    full, part = P // page, P % page
    need = [0 if n < 0 else -(-(P + n) // page) - full for n in lens]
    n_pages = case["groups"] * full + sum(need) + 3
    order = _perm(seed, n_pages)
    max_pages = full + max(1, max(need))
    k = torch.randn(n_pages, Hk, page, hd, generator=g, device=DEV, dtype=torch.float32).to(dt)
    v = torch.randn(n_pages, Hk, page, hd, generator=g, device=DEV, dtype=torch.float32).to(dt)
    q = (1.5 * torch.randn(B * S, Hq * hd, generator=g, device=DEV, dtype=torch.float32)).to(dt)
    rows, pos, at = [], [], 0
    for i in range(case["groups"]):
        shared = order[at:at + full]
        at += full
        first = None   # the page that holds the prefix's last, partial page of the first live sequence
        for b in range(gs[i], gs[i + 1]):
            if lens[b] < 0:
                rows.append([-1] * max_pages)
                pos += [-1] * S
                continue
            mine = order[at:at + need[b]]
            at += need[b]
            if part:
                if first is None:
                    first = mine[0]
                else:
                    k[mine[0], :, :part] = k[first, :, :part]
                    v[mine[0], :, :part] = v[first, :, :part]
            rows.append((shared + mine + [-1] * max_pages)[:max_pages])
            pos += [P + lens[b] - S + s for s in range(S)]
    # the prefix's pages stand in the table row of a live sequence of the group
    owner = [next((b for b in range(gs[i], gs[i + 1]) if lens[b] >= 0), gs[i]) for i in range(case["groups"])]
    plen = [P if lens[b] >= 0 else 0 for b in owner]
    return dict(case=case, q=q, k=k, v=v, table=torch.tensor(rows, dtype=torch.int32, device=DEV),
                pos=torch.tensor(pos, dtype=torch.int64, device=DEV),
                gstart=torch.tensor(gs, dtype=torch.int32, device=DEV),
                owner=torch.tensor(owner, dtype=torch.int32, device=DEV),
                plen=torch.tensor(plen, dtype=torch.int32, device=DEV), S=S)


def _pool(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    shape = (case["layers"], case["n_pages"], case["Hk"], case["page"], case["hd"])
    k = torch.empty(shape, device=DEV, dtype=dt)
    v = torch.empty(shape, device=DEV, dtype=dt)
    for i in range(case["layers"]):
        k[i] = torch.randn(shape[1:], generator=g, device=DEV)
        v[i] = torch.randn(shape[1:], generator=g, device=DEV)
    return k, v


def _fork_host(case, seed):
    """Lengths, tables and reference counts before the fork, and the fork's list."""
    page, n_src, n_dst = case["page"], case["n_src"], case["n_dst"]
    lens = [max(1, case["length"] - d) for d in _ints(case, seed, n_src, 0, min(page, case["length"] // 4))]
    held = -(-case["length"] // page)
    order, table, refs = _perm(seed, case["n_pages"]), [], [0] * case["n_pages"]
    for i, n in enumerate(lens):
        pages = order[i * held:i * held + -(-n // page)]
        for p in pages:
            refs[p] = 1
        table.append((pages + [-1] * (held + 1))[:held + 1])
    table += [[-1] * (held + 1) for _ in range(n_dst)]
    return lens + [0] * n_dst, table, refs, [i * n_src // n_dst for i in range(n_dst)], list(range(n_src, n_src + n_dst))


def _prep_fork(case, seed):
    k, v = _pool(case, seed)
    lens, table, refs, src, dst = _fork_host(case, seed)
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(case=case, k=k, v=v, table=torch.tensor(table, **i32), refs=torch.tensor(refs, **i32),
                lens=torch.tensor(lens, dtype=torch.int64, device=DEV), src=torch.tensor(src, **i32),
                dst=torch.tensor(dst, **i32), src_host=src, dst_host=dst, src_lens=[lens[s] for s in src])


def _compact_host(case, seed):
    n, ns = case["n_pages"], case["n_seqs"]
    live = sorted(_perm(seed, n)[:max(ns, min(n - 1, int(round(n * case["live"]))))])
    order = _perm(seed + 1, len(live))
    per, refs = -(-len(live) // ns), [0] * n
    table = []
    for i in range(ns):
        pages = [live[j] for j in order[i * per:(i + 1) * per]]
        if i and table[0][0] >= 0 and pages:
            pages[0] = table[0][0]   # a page that sequences share
        table.append((pages + [-1] * per)[:per])
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return table, refs


def _prep_compact(case, seed):
    k, v = _pool(case, seed)
    table, refs = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in _compact_host(case, seed))
    return dict(case=case, k=k, v=v, table0=table, refs0=refs, table=table.clone(), refs=refs.clone())


def _write_host(case):
    B, S, page, start = (case[x] for x in ("B", "S", "page", "start"))
    before, after = [], []
    for b in range(B):
        n = max(0, start - 3 * b)
        before.append(n)
        after.append(n + S)
    return before, after, max(-(-n // page) for n in after)


def _prep_write(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    B, S, Hq, Hk, hd, page = (case[x] for x in ("B", "S", "Hq", "Hk", "hd", "page"))
    before, after, held = _write_host(case)
    n_pages = B * held + 2
    order, rows, refs = _perm(seed, n_pages), [], [0] * n_pages
    for b in range(B):
        pages = order[b * held:b * held + -(-before[b] // page)]
        for p in pages:
            refs[p] = 1
        rows.append((pages + [-1] * held)[:held])
    pos = [before[b] + s for b in range(B) for s in range(S)]
    angle = torch.outer(torch.arange(max(after), dtype=torch.float64),
                        500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    i32 = dict(dtype=torch.int32, device=DEV)
    return dict(case=case, S=S, k=torch.randn(n_pages, Hk, page, hd, generator=g, device=DEV).to(dt),
                v=torch.randn(n_pages, Hk, page, hd, generator=g, device=DEV).to(dt),
                qkv=torch.randn(B * S, (Hq + 2 * Hk) * hd, generator=g, device=DEV).to(dt),
                rope=torch.stack([angle.cos(), angle.sin()], -1).float().to(DEV),
                pos=torch.tensor(pos, dtype=torch.int64, device=DEV), q_out=torch.empty(B * S, Hq * hd, device=DEV, dtype=dt),
                table0=torch.tensor(rows, **i32), refs0=torch.tensor(refs, **i32),
                lens0=torch.tensor(before, dtype=torch.int64, device=DEV), table=torch.tensor(rows, **i32),
                refs=torch.tensor(refs, **i32), lens=torch.tensor(before, dtype=torch.int64, device=DEV),
                seqs=torch.arange(B, **i32))


def _prep_mm(case, seed):
    g, dt = _gen(seed), TYPES[case["dtype"]]
    M, N, K = case["M"], case["N"], case["K"]
    x = torch.randn(M, K, generator=g, device=DEV)
    x[:, ::97] *= 8.0   # the few channels with large values that activations have
    w = (32.0 * torch.randn(N, K, generator=g, device=DEV)).round_().clamp_(-127, 127).to(torch.int8)
    s = ((0.5 + torch.rand(N, generator=g, device=DEV)) / (32.0 * math.sqrt(K))).to(torch.float16)
    r = torch.randn(M, N, generator=g, device=DEV).to(dt) if case["res"] else None
    return dict(case=case, x=x.to(dt), w=w, s=s, res=r)


def prepare(case, seed):
    return {"attn": _prep_attn, "fork": _prep_fork, "compact": _prep_compact, "write": _prep_write,
            "mm": _prep_mm}[case["op"]](case, seed)


# ----------------------------------------------------------------------------- plain forms
def _plain_attn(st):
    c, q, k, v, table, pos = st["case"], st["q"], st["k"], st["v"], st["table"], st["pos"]
    B, S, Hq, Hk, hd = c["B"], c["S"], c["Hq"], c["Hk"], c["hd"]
    G = Hq // Hk
    pages = table.clamp(min=0).long()
    T = pages.shape[1] * c["page"]
    kk = k[pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, T, hd).float()
    qq = q.view(B, S, Hk, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Hk, S * G, hd).float()
    s = (qq @ kk.transpose(-1, -2)) / math.sqrt(hd)
    seen = torch.arange(T, device=q.device)[None, None, :] <= pos.view(B, S, 1)
    s = s.view(B, Hk, S, G, T).masked_fill(~seen[:, None, :, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    vv = v[pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, T, hd).float()
    o = (p.view(B, Hk, S * G, T) @ vv).view(B, Hk, S, G, hd) / torch.where(l > 0, l, torch.ones_like(l))
    return o.permute(0, 2, 1, 3, 4).reshape(B * S, Hq * hd).to(q.dtype)


def _free_pages(refs):
    """Page numbers, the free ones first and in ascending order."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices


def _plain_fork(st):
    page, k, v, table, lens, refs = st["case"]["page"], st["k"], st["v"], st["table"], st["lens"], st["refs"]
    src, dst = st["src"].long(), st["dst"].long()
    # the last takes end: their pages lose a holder
    old = table[dst]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).flatten().to(torch.int32))
    # full pages of the source are shared, its last, partial page is copied into a free one
    t, n = table[src], lens[src]
    col = torch.arange(table.shape[1], device=t.device)[None, :]
    full = (n // page)[:, None]
    shared = col < full
    refs.index_add_(0, t.clamp(min=0).flatten().long(), shared.flatten().to(torch.int32))
    free, used = _free_pages(refs), 0
    new = torch.where(shared, t, torch.full_like(t, -1))
    for i, length in enumerate(st["src_lens"]):
        part, last = length % page, length // page
        if part:
            to, at = free[used], t[i, last].long()
            used += 1
            k[:, to, :, :part] = k[:, at, :, :part]
            v[:, to, :, :part] = v[:, at, :, :part]
            new[i, last] = to.to(torch.int32)
    refs[free[:used]] = 1
    table[dst] = new
    lens[dst] = n
    return k, v, table, lens, refs


def _plain_compact(st):
    k, v, table, refs = st["k"], st["v"], st["table"], st["refs"]
    table.copy_(st["table0"])
    refs.copy_(st["refs0"])
    at = torch.arange(refs.numel(), device=refs.device)
    live = refs > 0
    n_live = live.sum()
    src, dst = at[live & (at >= n_live)], at[~live & (at < n_live)]
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    moved = at.clone()
    moved[src] = dst
    table.copy_(torch.where(table >= 0, moved[table.clamp(min=0).long()].to(torch.int32), table))
    refs[dst] = refs[src]
    refs[src] = 0
    return k, v, table, refs, n_live.to(torch.int32).reshape(1)


def _plain_write(st):
    c, k, v, table, lens, refs = st["case"], st["k"], st["v"], st["table"], st["lens"], st["refs"]
    B, S, Hq, Hk, hd, page = c["B"], c["S"], c["Hq"], c["Hk"], c["hd"], c["page"]
    table.copy_(st["table0"])
    refs.copy_(st["refs0"])
    lens.copy_(st["lens0"])
    # pages for S more positions of every sequence
    have, want = (lens + page - 1) // page, (lens + S + page - 1) // page
    first = torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    free = _free_pages(refs)
    to = free[(first[:, None] + col - have[:, None]).clamp(0, free.numel() - 1)]
    table.copy_(torch.where(fresh, to.to(torch.int32), table))
    refs.index_add_(0, to.flatten(), fresh.flatten().to(torch.int32))
    lens += S
    # rotate q and k by their positions' angles, write k and v into their slots
    pos = st["pos"]
    x = st["qkv"].view(B * S, Hq + 2 * Hk, hd)
    rot = x[:, :Hq + Hk].float().view(B * S, Hq + Hk, hd // 2, 2)
    cs, sn = st["rope"][pos][:, None, :, 0], st["rope"][pos][:, None, :, 1]
    y = torch.stack([rot[..., 0] * cs - rot[..., 1] * sn, rot[..., 1] * cs + rot[..., 0] * sn], -1).view(B * S, Hq + Hk, hd)
    y = y.to(k.dtype)
    seq = torch.arange(B, device=pos.device).repeat_interleave(S)
    slot = table[seq, pos // page].long()
    k[slot, :, pos % page] = y[:, Hq:]
    v[slot, :, pos % page] = x[:, Hq + Hk:]
    st["q_out"].copy_(y[:, :Hq].reshape(B * S, Hq * hd))
    return st["q_out"], k, v, table, lens, refs


def _plain_mm(st):
    x, w, s, res = st["x"].float(), st["w"], st["s"].float(), st["res"]
    amax = x.abs().amax(-1, keepdim=True)
    # x * 127 is exact in 32 bits, so one division decides the rounding
    q = torch.where(amax > 0, torch.round(x * 127.0 / amax), torch.zeros_like(x))
    y = (q @ w.float().t()) * (amax / 127.0) * s
    if st["case"]["silu"]:
        a, b = y.chunk(2, -1)
        y = a / (1.0 + torch.exp(-a)) * b
    if res is not None:
        y = y + res.float()
    return y.to(st["x"].dtype)


# ----------------------------------------------------------------------------- the framework's calls
def _own_attn(st):
    from estudiocanciones_b200 import kernels
    return kernels.prefix_attn(st["q"], st["k"], st["v"], st["table"], st["pos"], st["gstart"], st["owner"], st["plen"],
                               st["S"])


def _own_fork(st):
    from estudiocanciones_b200 import kernels
    kernels.pages_free(st["table"], st["lens"], st["refs"], st["dst"])
    kernels.pages_fork(st["k"], st["v"], st["table"], st["lens"], st["refs"], st["src"], st["dst"])
    return st["k"], st["v"], st["table"], st["lens"], st["refs"]


def _own_compact(st):
    from estudiocanciones_b200 import kernels
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])
    n_live = kernels.pages_compact(st["k"], st["v"], st["table"], st["refs"])
    return st["k"], st["v"], st["table"], st["refs"], n_live


def _own_write(st):
    from estudiocanciones_b200 import kernels
    c = st["case"]
    st["table"].copy_(st["table0"])
    st["refs"].copy_(st["refs0"])
    st["lens"].copy_(st["lens0"])
    kernels.pages_grow(st["table"], st["lens"], st["refs"], c["page"], st["seqs"], c["S"])
    kernels.rope_pages(st["qkv"], st["rope"], st["pos"], st["q_out"], st["k"], st["v"], st["table"], c["S"], c["Hq"],
                       c["Hk"])
    return st["q_out"], st["k"], st["v"], st["table"], st["lens"], st["refs"]


def _own_mm(st):
    from estudiocanciones_b200 import kernels
    return kernels.int8_mm_a8(st["x"], st["w"], st["s"], st["res"], silu=st["case"]["silu"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "fork": _own_fork, "compact": _own_compact, "write": _own_write,
                "mm": _own_mm}[op](state)
    return {"attn": _plain_attn, "fork": _plain_fork, "compact": _plain_compact, "write": _plain_write,
            "mm": _plain_mm}[op](state)


# ----------------------------------------------------------------------------- cost
def work(case):
    op = case["op"]
    if op == "mm":
        M, N, K = case["M"], case["N"], case["K"]
        out = M * (N // 2 if case["silu"] else N)
        return {"bytes": 2 * M * K + N * K + 2 * N + 2 * out + (2 * out if case["res"] else 0), "flops": 2 * M * N * K}
    row = 2 * 2 * case["Hk"] * case["hd"]   # K and V of one position
    if op == "attn":
        B, S, Hq, hd, P = (case[x] for x in ("B", "S", "Hq", "hd", "prefix"))
        mean = (S + case["own_max"]) / 2 if case["ragged"] else case["own_max"]
        live = B - 1 if case["pad"] and B > 1 else B
        return {"bytes": int(row * (case["groups"] * P + live * mean) + 4 * B * S * Hq * hd),
                "flops": int(4 * live * S * Hq * hd * (P + mean))}
    if op == "fork":
        part = case["length"] % case["page"]
        return {"bytes": 2 * case["n_dst"] * case["layers"] * row * part + 8 * case["n_pages"], "flops": 0}
    if op == "compact":
        n, f = case["n_pages"], case["live"]
        return {"bytes": int(2 * n * f * (1 - f) * case["layers"] * row * case["page"]) + 8 * n, "flops": 0}
    R = case["B"] * case["S"]
    qkv = 2 * (case["Hq"] + 2 * case["Hk"]) * case["hd"]
    return {"bytes": 2 * R * qkv + 4 * case["S"] * case["hd"], "flops": 3 * R * (case["Hq"] + case["Hk"]) * case["hd"]}


# ----------------------------------------------------------------------------- definitions in 64 bits
def _exact_attn(case, seed):
    st = _prep_attn(case, seed)
    B, S, Hq, Hk, hd, page = (case[x] for x in ("B", "S", "Hq", "Hk", "hd", "page"))
    table, pos = st["table"].tolist(), st["pos"].tolist()
    q = st["q"].double().view(B * S, Hk, Hq // Hk, hd)
    out = torch.zeros(B * S, Hk, Hq // Hk, hd, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = pos[b * S + S - 1] + 1
        if n <= 0:
            continue
        ids = table[b][:-(-n // page)]
        kk = torch.cat([st["k"][p] for p in ids], 1)[:, :n].double()   # [Hk, n, hd]
        vv = torch.cat([st["v"][p] for p in ids], 1)[:, :n].double()
        for s in range(S):
            m = pos[b * S + s] + 1
            if m > 0:
                z = torch.einsum("hgd,hnd->hgn", q[b * S + s], kk[:, :m]) * hd ** -0.5
                out[b * S + s] = torch.einsum("hgn,hnd->hgd", torch.softmax(z, -1), vv[:, :m])
    return out.view(B * S, Hq * hd)


def _exact_fork(case, seed):
    k, v = _pool(case, seed)
    lens, table, refs, src, dst = _fork_host(case, seed)
    page = case["page"]
    for a, b in zip(src, dst):
        lens[b] = lens[a]
        for j in range(lens[a] // page):
            table[b][j] = table[a][j]
            refs[table[a][j]] += 1
    for a, b in zip(src, dst):
        j, part = divmod(lens[a], page)
        if part:
            p = refs.index(0)
            refs[p], table[b][j] = 1, p
            k[:, p, :, :part] = k[:, table[a][j], :, :part]
            v[:, p, :, :part] = v[:, table[a][j], :, :part]
    return (k, v, torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(lens, device=DEV),
            torch.tensor(refs, dtype=torch.int32, device=DEV))


def _exact_compact(case, seed):
    k, v = _pool(case, seed)
    table, refs = _compact_host(case, seed)
    n_live = sum(r > 0 for r in refs)
    holes = [p for p in range(n_live) if refs[p] == 0]
    high = [p for p in range(n_live, len(refs)) if refs[p] > 0]
    to = dict(zip(high, holes))
    for a, b in to.items():
        k[:, b], v[:, b] = k[:, a], v[:, a]
        refs[b], refs[a] = refs[a], 0
    table = [[to.get(p, p) for p in row] for row in table]
    i32 = dict(dtype=torch.int32, device=DEV)
    return k, v, torch.tensor(table, **i32), torch.tensor(refs, **i32), torch.tensor([n_live], **i32)


def _exact_write(case, seed):
    st = _prep_write(case, seed)
    B, S, Hq, Hk, hd, page = (case[x] for x in ("B", "S", "Hq", "Hk", "hd", "page"))
    table, refs, lens = st["table0"].tolist(), st["refs0"].tolist(), st["lens0"].tolist()
    pages, slots = [], []
    for b in range(B):
        for j in range(-(-lens[b] // page), -(-(lens[b] + S) // page)):
            p = refs.index(0)
            refs[p], table[b][j] = 1, p
        for n in range(lens[b], lens[b] + S):
            pages.append(table[b][n // page])
            slots.append(n % page)
        lens[b] += S
    pages, slots = torch.tensor(pages, device=DEV), torch.tensor(slots, device=DEV)
    turn = torch.view_as_complex(st["rope"].double().contiguous())[st["pos"]]
    x = st["qkv"].double().view(B * S, Hq + 2 * Hk, hd)
    z = torch.view_as_complex(x[:, :Hq + Hk].reshape(B * S, Hq + Hk, hd // 2, 2).contiguous()) * turn[:, None]
    y = torch.view_as_real(z).reshape(B * S, Hq + Hk, hd)
    k, v = st["k"].double(), st["v"].double()
    k[pages, :, slots] = y[:, Hq:]
    v[pages, :, slots] = x[:, Hq + Hk:]
    i32 = dict(dtype=torch.int32, device=DEV)
    return (y[:, :Hq].reshape(B * S, Hq * hd), k, v, torch.tensor(table, **i32), torch.tensor(lens, device=DEV),
            torch.tensor(refs, **i32))


def _exact_mm(case, seed):
    st = _prep_mm(case, seed)
    x = st["x"].double()
    top = x.abs().max(dim=-1).values[:, None]
    q = (x * 127 / top.clamp(min=1e-300)).round()
    y = torch.mm(q, st["w"].double().T) * (top / 127) * st["s"].double()[None, :]
    if case["silu"]:
        half = y.shape[1] // 2
        y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
    return y if st["res"] is None else y + st["res"].double()


def exact(case, seed):
    return {"attn": _exact_attn, "fork": _exact_fork, "compact": _exact_compact, "write": _exact_write,
            "mm": _exact_mm}[case["op"]](case, seed)
