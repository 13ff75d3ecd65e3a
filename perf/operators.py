"""Cases for the paged KV cache operators: append with rotation, paged attention, shared-prefix attention.

Every case names one call that a serving program makes on a cache of 128-wide heads held in pages.
``run`` computes it in plain torch operations (``own`` false) or through the package (``own`` true).

Conventions shared by the three operators:
  k_pages, v_pages  [n_pages, Hkv, page, 128]; "nhd" cases hold them as [n_pages, page, Hkv, 128]
  block_table       int32 [B, max_pages], -1 where a sequence holds no page
  seq_lens          int32 [B], tokens of a sequence in the cache, the new ones included
  q_lens            int32 [B], how many of the Tq rows of a sequence are live
  row t of sequence b is the token at position seq_lens[b] - q_lens[b] + t
Cache slots that hold no token are NaN: pages are recycled, so nothing may be assumed about them.
"""
import math

import torch

own = False

D = 128
BLOCK = 128
DEV = "cuda"


def _case(name, op, B, Hq, Hkv, Tq, lo, hi, page, dtype, layout="hnd", window=0, glob=0, prefix=0,
          rot=128, interleaved=False, ragged=False):
    """lo..hi: tokens of a sequence in the cache after this call (behind the prefix, if there is
    one), spread evenly over the batch.  ragged: q_lens spread over 0..Tq instead of Tq for all."""
    return dict(name=name, op=op, B=B, Hq=Hq, Hkv=Hkv, Tq=Tq, lo=lo, hi=hi, page=page, dtype=dtype,
                layout=layout, window=window, glob=glob, prefix=prefix, rot=rot,
                interleaved=interleaved, ragged=ragged)


def listed():
    return [
        # One user, one token: latency is all there is.
        _case("append_one_token", "append", 1, 16, 16, 1, 701, 701, 64, "bf16"),
        # A full decode batch, grouped heads, a half-width interleaved rotation, token-major pages.
        _case("append_batch", "append", 256, 32, 8, 1, 17, 8000, 16, "fp16", layout="nhd", rot=64,
              interleaved=True),
        # The prompts of the headline prefill (B=2, H=16, T=8192) go into the cache, padded batch.
        _case("append_prefill", "append", 2, 16, 16, 8192, 8192, 8300, 64, "bf16", ragged=True),
        # One user, a short odd context.
        _case("decode_one", "paged", 1, 16, 16, 1, 777, 777, 64, "fp16"),
        # A usual serving batch, ragged lengths, small pages.
        _case("decode_batch", "paged", 32, 32, 8, 1, 333, 8192, 16, "bf16"),
        # Long contexts: the cache is far larger than L2.
        _case("decode_long", "paged", 8, 32, 8, 1, 100001, 131072, 64, "fp16", layout="nhd"),
        # The framework's window + global-prefix rows, continued token by token.
        _case("decode_window", "paged", 16, 32, 8, 1, 20011, 32768, 128, "bf16", window=8, glob=4),
        # Checking five drafted tokens at once, odd group of seven heads.
        _case("verify_five", "paged", 24, 28, 4, 5, 1000, 4099, 32, "fp16", ragged=True),
        # A chunk of a long prompt against what is cached already.
        _case("prefill_chunk", "paged", 2, 32, 8, 512, 4000, 8192, 64, "bf16"),
        # Few answers to one short shared prompt.
        _case("shared_small", "shared", 8, 16, 2, 1, 1, 64, 16, "bf16", prefix=1024),
        # Many users behind a long common document.
        _case("shared_long", "shared", 64, 32, 8, 1, 100, 1000, 64, "bf16", prefix=32768),
        # A wide batch behind a system prompt: the shared part is bound by the tensor cores.
        _case("shared_wide", "shared", 256, 32, 8, 1, 1, 511, 32, "fp16", layout="nhd",
              prefix=8192),
    ]


# (Hq, Hkv): equal heads as in the prefill configurations, and the usual and odd group sizes.
_HEADS = [(16, 16), (32, 32), (32, 8), (16, 2), (8, 1), (6, 2), (28, 4), (20, 4), (12, 12), (32, 2)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    while True:
        op = rng.choice(["append", "paged", "paged", "shared"])
        Hq, Hkv = rng.choice(_HEADS)
        B = _log(rng, 1, 256)
        Tq = 1 if rng.random() < 0.5 else _log(rng, 2, 8192 if op == "append" else 512)
        page = rng.choice([16, 32, 64, 128, 256])
        rot, inter, window, glob, prefix = 128, False, 0, 0, 0
        hi = _log(rng, max(Tq, 1), 131072)
        if op == "append":
            rot, inter = rng.choice([128, 128, 64, 32]), rng.random() < 0.3
            hi = max(Tq, hi // 8)
        elif op == "paged":
            if rng.random() < 0.3:
                window, glob = _log(rng, 1, 32), rng.choice([0, 1, 4])
        else:
            prefix = max(1, _log(rng, 16, 32768) // page) * page
            hi = max(Tq, min(hi, 2048))
        lo = rng.randint(Tq, hi) if rng.random() < 0.8 else hi
        c = _case("", op, B, Hq, Hkv, Tq, lo, hi, page, rng.choice(["fp16", "bf16"]),
                  rng.choice(["hnd", "hnd", "nhd"]), window, glob, prefix, rot, inter,
                  Tq > 1 and rng.random() < 0.5)
        del c["name"]
        held = (B * hi + prefix) * Hkv            # cached tokens x heads
        scored = B * Tq * (hi + prefix) * Hq      # scores of the plain form
        rows = B * Tq * (Hq + 2 * Hkv)
        if held <= 8 * 131072 * 8 // 2 and rows <= 800_000 and (op == "append" or scored <= 1.9e8):
            return c


def _lens(c):
    """Lengths of the sequences, own tokens only, in a fixed order: even steps from lo to hi."""
    B = c["B"]
    return [c["hi"] if B == 1 else c["lo"] + (c["hi"] - c["lo"]) * b // (B - 1) for b in range(B)]


def _live(c):
    """Live rows of the sequences (the last one may be empty in a padded batch)."""
    B, Tq = c["B"], c["Tq"]
    if not c["ragged"] or B == 1:
        return [Tq] * B
    return [max(0, Tq - Tq * b // B - (b % 2)) for b in range(B)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
    B, Hq, Hkv, Tq, ps, pre = c["B"], c["Hq"], c["Hkv"], c["Tq"], c["page"], c["prefix"]
    order = torch.randperm(B, generator=gc)
    own_len = torch.tensor(_lens(c))[order]
    q_lens = torch.tensor(_live(c))[torch.randperm(B, generator=gc)]
    lens = own_len + pre
    # Pages in random order, some never used; the shared prefix's pages come first in every row.
    npre = pre // ps
    own_pages = (own_len + ps - 1) // ps
    n_pages = npre + int(own_pages.sum()) + 3
    ids = torch.randperm(n_pages, generator=gc)
    width = npre + int(own_pages.max()) + 1
    ar = torch.arange(width - npre)
    base = npre + torch.cumsum(own_pages, 0) - own_pages
    held = ar[None, :] < own_pages[:, None]
    table = torch.full((B, width), -1, dtype=torch.int64)
    table[:, :npre] = ids[:npre]
    table[:, npre:] = torch.where(held, ids[(base[:, None] + ar).clamp(max=n_pages - 1)], -1)
    # Tokens held: all of them for attention, those before the new ones for an append.
    before = lens - (q_lens if c["op"] == "append" else 0)
    col = torch.arange(width)
    count = (before[:, None] - col * ps).clamp(0, ps)
    fill = torch.zeros(n_pages + 1, dtype=torch.int64)
    fill[torch.where(table < 0, n_pages, table)] = torch.where(table < 0, 0, count)
    empty = (torch.arange(ps) >= fill[:n_pages, None]).to(DEV)
    pages = []
    for _ in range(2):
        if c["layout"] == "nhd":
            t = torch.randn(n_pages, ps, Hkv, D, generator=g, device=DEV, dtype=dt)
            t.masked_fill_(empty[:, :, None, None], float("nan"))
            t = t.permute(0, 2, 1, 3)
        else:
            t = torch.randn(n_pages, Hkv, ps, D, generator=g, device=DEV, dtype=dt)
            t.masked_fill_(empty[:, None, :, None], float("nan"))
        pages.append(t)
    s = dict(case=dict(c), k_pages=pages[0], v_pages=pages[1],
             block_table=table.to(DEV, torch.int32), seq_lens=lens.to(DEV, torch.int32),
             q_lens=q_lens.to(DEV, torch.int32) if c["ragged"] else None, n_pages=n_pages)
    if c["op"] == "append":
        # q, k, v as a projection leaves them: one [B, Tq, heads * 128] tensor, seen by head.
        qkv = torch.randn(B, Tq, Hq + 2 * Hkv, D, generator=g, device=DEV, dtype=dt)
        s["q"], s["k"], s["v"] = [t.transpose(1, 2) for t in qkv.split([Hq, Hkv, Hkv], 2)]
        i = torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64)
        s["inv_freq"] = 10000.0 ** (-2.0 * i / c["rot"])
    else:
        s["q"] = 2 * torch.randn(B, Hq, Tq, D, generator=g, device=DEV, dtype=dt)
    return s


def run(state):
    s, c = state, state["case"]
    if own:
        import usagi_b200 as ub
        cache = (s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"])
        if c["op"] == "append":
            q = ub.paged_kv_append(*cache, s["k"], s["v"], q=s["q"], q_lens=s["q_lens"],
                                   inv_freq=s["inv_freq"], interleaved=c["interleaved"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if c["op"] == "paged":
            o, lse = ub.paged_attn_fwd(s["q"], *cache, q_lens=s["q_lens"],
                                       window=c["window"] or None, global_blocks=c["glob"])
        else:
            o, lse = ub.shared_prefix_attn_fwd(s["q"], *cache, prefix_len=c["prefix"],
                                               q_lens=s["q_lens"])
        return {"o": o, "lse": lse}
    return {"append": _plain_append, "paged": _plain_paged, "shared": _plain_shared}[c["op"]](s)


# ------------------------------------------------------------------------------------------------
# Plain forms
# ------------------------------------------------------------------------------------------------
def _positions(s):
    """(positions [B, Tq], live [B, Tq]) of the new rows."""
    Tq = s["q"].shape[2]
    t = torch.arange(Tq, device=DEV)
    sl = s["seq_lens"].long()
    ql = torch.full_like(sl, Tq) if s["q_lens"] is None else s["q_lens"].long()
    pos = sl[:, None] - ql[:, None] + t
    return pos, (t < ql[:, None]) & (pos >= 0)


def _rotate(x, cos, sin, rot, interleaved):
    x = x.float()
    a, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        x0, x1 = a[..., 0::2], a[..., 1::2]
        y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    else:
        x0, x1 = a[..., :rot // 2], a[..., rot // 2:]
        y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    return torch.cat([y, rest], -1)


def _plain_append(s):
    c, kp, vp = s["case"], s["k_pages"], s["v_pages"]
    pos, live = _positions(s)
    angle = pos.double()[..., None] * s["inv_freq"]          # 64 bits: far positions
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    rot = (cos, sin, c["rot"], c["interleaved"])
    q = torch.where(live[:, None, :, None], _rotate(s["q"], *rot), 0.0).to(s["q"].dtype)
    k = _rotate(s["k"], *rot).to(kp.dtype)
    # Padding rows repeat the last live row of their sequence, so every row may be written.
    B, Tq = pos.shape
    n = live.sum(1)
    t = torch.minimum(torch.arange(Tq, device=DEV)[None, :], (n[:, None] - 1).clamp(min=0))
    at = torch.gather(pos, 1, t).clamp(min=0)
    at = torch.minimum(at, (s["seq_lens"].long()[:, None] - 1).clamp(min=0))
    page = torch.gather(s["block_table"].long(), 1, at // c["page"])
    slot = at % c["page"]
    b = torch.arange(B, device=DEV)[:, None]
    for pages, new in ((kp, k), (vp, s["v"])):
        keep = pages[page, :, slot]
        pages[page, :, slot] = torch.where(n[:, None, None, None] > 0,
                                           new.transpose(1, 2)[b, t], keep)
    return {"q": q, "k_pages": kp, "v_pages": vp}


def _gather(pages, table, lens, first):
    """Tokens `first`.. of every sequence as [B, Hkv, L, 128] in 32 bits, 0 where there is none."""
    B, W = table.shape
    x = pages[table.long().clamp(min=0)]                     # [B, W, Hkv, page, 128]
    x = x.permute(0, 2, 1, 3, 4).reshape(B, x.shape[2], -1, D).float()
    j = first + torch.arange(x.shape[2], device=DEV)
    return x.masked_fill_((j >= lens[:, None])[:, None, :, None], 0.0)


def _allowed(s, j):
    """Which keys j each row may see: [B, 1, 1, Tq, len(j)]."""
    c = s["case"]
    pos, live = _positions(s)
    p = pos[..., None]
    ok = live[..., None] & (j <= p)
    if c["window"]:
        ok &= (j // BLOCK < c["glob"]) | (j // BLOCK > p // BLOCK - c["window"])
    return ok[:, None, None]


def _finish(s, scores, values):
    """Softmax over the joined parts; scores [B, Hkv, G, Tq, n], values(p, i) the i-th product."""
    dt = s["q"].dtype
    m = scores[0].amax(-1, keepdim=True)
    for x in scores[1:]:
        m = torch.maximum(m, x.amax(-1, keepdim=True))
    m = torch.where(m.isinf(), 0.0, m)
    p = [(x - m).exp_() for x in scores]
    total = sum(x.sum(-1, keepdim=True) for x in p)
    o = sum(values(x, i) for i, x in enumerate(p)) / torch.where(total > 0, total, 1.0)
    B, Hkv, G, Tq, _ = o.shape
    lse = m + total.log()
    return {"o": o.reshape(B, Hkv * G, Tq, D).to(dt), "lse": lse.reshape(B, Hkv * G, Tq)}


def _plain_paged(s):
    return _plain_attn(s, 0)


def _plain_shared(s):
    return _plain_attn(s, s["case"]["prefix"])


def _plain_attn(s, pre):
    c = s["case"]
    B, Hq, Tq, _ = s["q"].shape
    Hkv, ps = c["Hkv"], c["page"]
    G = Hq // Hkv
    q = s["q"].float().reshape(B, Hkv, G * Tq, D) / math.sqrt(D)
    own_table = s["block_table"][:, pre // ps:]
    k = _gather(s["k_pages"], own_table, s["seq_lens"], pre)
    v = _gather(s["v_pages"], own_table, s["seq_lens"], pre)
    n = k.shape[2]
    own_scores = (q @ k.transpose(-1, -2)).reshape(B, Hkv, G, Tq, n)
    j = pre + torch.arange(n, device=DEV)
    own_scores = own_scores.masked_fill(~_allowed(s, j), float("-inf"))
    if not pre:
        return _finish(s, [own_scores], lambda p, i: (p.reshape(B, Hkv, -1, n) @ v).reshape(
            B, Hkv, G, Tq, D))
    # The prefix once: its keys against the rows of the whole batch, [Hkv, B * G * Tq, prefix].
    shared = s["block_table"][:1, :pre // ps]
    kp = _gather(s["k_pages"], shared, torch.full_like(s["seq_lens"][:1], pre), 0)[0]
    vp = _gather(s["v_pages"], shared, torch.full_like(s["seq_lens"][:1], pre), 0)[0]
    rows = q.transpose(0, 1).reshape(Hkv, -1, D)
    x = (rows @ kp.transpose(-1, -2)).reshape(Hkv, B, G, Tq, pre).transpose(0, 1)
    x = x.masked_fill(~_allowed(s, torch.arange(pre, device=DEV)), float("-inf"))

    def values(p, i):
        if i == 0:
            return (p.reshape(B, Hkv, -1, n) @ v).reshape(B, Hkv, G, Tq, D)
        y = p.transpose(0, 1).reshape(Hkv, -1, pre) @ vp
        return y.reshape(Hkv, B, G, Tq, D).transpose(0, 1)

    return _finish(s, [own_scores, x], values)


# ------------------------------------------------------------------------------------------------
# Work and exact values
# ------------------------------------------------------------------------------------------------
def _blocks_seen(c, pos):
    """Blocks of 128 keys that the row at `pos` sees under window + global blocks."""
    i = pos // BLOCK
    first = max(0, i - c["window"] + 1)
    return min(c["glob"], first), first, i


def work(case):
    c = case
    Hq, Hkv, Tq, pre = c["Hq"], c["Hkv"], c["Tq"], c["prefix"]
    lens = _lens(c)
    live = sum(_live(c))
    if c["op"] == "append":
        per = (Hq + 2 * Hkv) * D
        # Every live row is read and written; padding rows of q are written as zeros.
        return {"bytes": 4.0 * per * live + 2.0 * Hq * D * (c["B"] * Tq - live),
                "flops": 3.0 * (Hq + Hkv) * c["rot"] * live}
    rows = live / c["B"]                 # q_lens are dealt by the seed: their mean
    read = scored = 0.0
    for n in lens:
        n += pre
        if c["window"]:
            g, f, i = _blocks_seen(c, max(0, n - int(rows) if Tq > 1 else n - 1))
            read += min(n, g * BLOCK + n - f * BLOCK)
            scored += rows * min(n, g * BLOCK + n - f * BLOCK)
        else:
            read += n - pre
            scored += rows * (n - (rows - 1) / 2)
    read += pre
    qo = 2.0 * D * 2 * Hq * Tq * c["B"] + 4.0 * Hq * Tq * c["B"]
    return {"bytes": 4.0 * D * Hkv * read + qo, "flops": 4.0 * D * Hq * scored}


def exact(case, seed):
    """The definition in 64 bits, one sequence at a time."""
    c = case
    s = prepare(case, seed)
    B, Hq, Hkv, Tq, ps = c["B"], c["Hq"], c["Hkv"], c["Tq"], c["page"]
    lens = s["seq_lens"].tolist()
    live = s["q_lens"].tolist() if s["q_lens"] is not None else [Tq] * B
    table = s["block_table"].long()
    if c["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        q = torch.zeros(B, Hq, Tq, D, device=DEV, dtype=torch.float64)
        for b in range(B):
            n = live[b]
            at = torch.arange(lens[b] - n, lens[b], device=DEV)
            turn = torch.polar(torch.ones(n, c["rot"] // 2, device=DEV, dtype=torch.float64),
                               at[:, None].double() * s["inv_freq"])

            def rotated(x):
                x = x.double()
                a = x[..., :c["rot"]]
                pairs = a.unflatten(-1, (-1, 2)) if c["interleaved"] else \
                    a.unflatten(-1, (2, -1)).transpose(-1, -2)
                y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
                y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
                return torch.cat([y, x[..., c["rot"]:]], -1)

            q[b, :, :n] = rotated(s["q"][b, :, :n])
            page, slot = table[b, at // ps], at % ps
            kp[page, :, slot] = rotated(s["k"][b, :, :n]).transpose(0, 1)
            vp[page, :, slot] = s["v"][b, :, :n].double().transpose(0, 1)
        return {"q": q, "k_pages": kp, "v_pages": vp}
    o = torch.zeros(B, Hq, Tq, D, device=DEV, dtype=torch.float64)
    lse = torch.full((B, Hq, Tq), float("-inf"), device=DEV, dtype=torch.float64)
    for b in range(B):
        n, L = live[b], lens[b]
        if n == 0:
            continue
        at = torch.arange(L - n, L, device=DEV)
        j = torch.arange(L, device=DEV)
        seen = j <= at[:, None]
        if c["window"]:
            seen &= ((at[:, None] // BLOCK - j // BLOCK) < c["window"]) | (j < c["glob"] * BLOCK)
        used = j[seen.any(0)]
        hide = ~seen[:, used]
        page, slot = table[b, used // ps], used % ps
        for h in range(Hkv):
            k = s["k_pages"][page, h, slot].double()
            v = s["v_pages"][page, h, slot].double()
            hs = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            x = torch.einsum("gtd,jd->gtj", s["q"][b, hs, :n].double(), k) * D ** -0.5
            x.masked_fill_(hide, float("-inf"))
            lse[b, hs, :n] = torch.logsumexp(x, -1)
            o[b, hs, :n] = torch.einsum("gtj,jd->gtd", torch.softmax(x, -1), v)
    return {"o": o, "lse": lse}
