"""64-bit restatement of the paged-cache operators for the tests, with error bounds.

Kept apart from the package and from the other oracle: attention here is over a cache that is
rebuilt token by token from the page table, one sequence and one head at a time.

Bounds.  With u = half a step of the operands' type, a row's weights p_j (summing to 1) and values
v_j, let A = sum_j p_j |v_j|.  The kernel rounds each p_j to that type (u A), stores o in its own
type (u_out |o|), and works in 32 bits otherwise: a score of 128 products is off by at most
128 * 2^-24 * S, S = scale * max_j sum_i |q_i k_ji| (the order of the sum does not matter), a
weight by that much again in relative terms, plus 2^-22 for the exponential and n * 2^-24 for sums
over n keys; each enters o twice, through the numerator and the sum.  lse is off by the same
relative error of the sum once, plus a few 32-bit steps of its own size.
"""
import math

import torch

D = 128


class Cache:
    """A paged cache with NaN in every slot that holds no token, and its dense copy."""

    def __init__(self, lens, Hkv, page, dtype, seed, device, layout="hnd", extra_pages=2,
                 prefix=0, width_extra=1):
        g = torch.Generator().manual_seed(seed)
        self.page, self.dtype, self.device = page, dtype, device
        B = len(lens)
        npre = prefix // page
        per = [max(0, -(-n // page) - npre) for n in lens]
        n_pages = npre + sum(per) + extra_pages
        ids = torch.randperm(n_pages, generator=g)
        width = npre + max(per) + width_extra
        table = torch.full((B, width), -7, dtype=torch.int32)
        at = npre
        for b in range(B):
            table[b, :npre] = ids[:npre]
            table[b, npre:npre + per[b]] = ids[at:at + per[b]]
            at += per[b]
        shape = (n_pages, page, Hkv, D) if layout == "nhd" else (n_pages, Hkv, page, D)
        self.pages = []
        for _ in range(2):
            x = torch.randn(shape, generator=g).to(dtype)
            x = x.transpose(1, 2) if layout == "nhd" else x
            used = torch.zeros(n_pages, page, dtype=torch.bool)
            for b, n in enumerate(lens):
                for j in range(-(-n // page)):
                    used[table[b, j], :max(0, min(page, n - j * page))] = True
            for s in range(2):  # keeps the layout
                x[(~used)[:, None, :, None].expand_as(x)] = float("nan")
            self.pages.append(x)
        self.table, self.lens = table, list(lens)

    def dense(self, b, n, which):
        """Tokens 0..n-1 of sequence b: [Hkv, n, 128] in 64 bits."""
        x = self.pages[which]
        j = torch.arange(n)
        return x[self.table[b, j // self.page].long(), :, j % self.page].double().transpose(0, 1)

    def to(self, device):
        """(k_pages, v_pages, block_table, seq_lens) on a device, strides kept."""
        return (*(p.to(device) for p in self.pages), self.table.to(device),
                torch.tensor(self.lens, dtype=torch.int32, device=device))


def attention(q, cache, q_lens=None, window=0, glob=0, scale=None, out_dtype=None):
    """(o, lse, bound_o, bound_lse) in 64 bits for q [B, Hq, Tq, 128] on the CPU."""
    B, Hq, Tq, _ = q.shape
    Hkv = cache.pages[0].shape[1]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(cache.dtype).eps / 2
    u_out = torch.finfo(out_dtype or q.dtype).eps / 2
    o = torch.zeros(B, Hq, Tq, D, dtype=torch.float64)
    lse = torch.full((B, Hq, Tq), -math.inf, dtype=torch.float64)
    bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        L = cache.lens[b]
        n = Tq if q_lens is None else q_lens[b]
        if L == 0 or n == 0:
            continue
        k, v = cache.dense(b, L, 0), cache.dense(b, L, 1)
        j = torch.arange(L)
        for t in range(n):
            p = L - n + t
            if p < 0:
                continue
            seen = j <= p
            if window:
                seen &= (j // 128 < glob) | (j // 128 > p // 128 - window)
            qh = q[b, :, t].double().reshape(Hkv, G, D)
            x = scale * qh @ k[:, seen].transpose(1, 2)
            w = torch.softmax(x, -1)
            rows = slice(0, Hq)
            o[b, rows, t] = (w @ v[:, seen]).reshape(Hq, D)
            lse[b, rows, t] = torch.logsumexp(x, -1).reshape(Hq)
            A = (w @ v[:, seen].abs()).reshape(Hq, D)
            S = scale * (qh.abs() @ k[:, seen].abs().transpose(1, 2)).amax(-1).reshape(Hq)
            rel = 128 * 2.0 ** -24 * S + 2.0 ** -22 + int(seen.sum()) * 2.0 ** -24
            bo[b, rows, t] = u * A + u_out * o[b, rows, t].abs() + 2 * rel[:, None] * A
            # fp16 stores below its smallest normal value lose a fixed step instead
            bo[b, rows, t] += torch.finfo(out_dtype or q.dtype).tiny * 2 * u_out
            bl[b, rows, t] = rel + 4 * 2.0 ** -24 * (lse[b, rows, t].abs() + 1)
    return o, lse, bo, bl


def check_attention(o, lse, want):
    ro, rl, bo, bl = want
    o, lse = o.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isinf(rl), torch.isinf(lse))
    assert torch.isfinite(o).all()
    over = (o - ro).abs() / bo.clamp(min=1e-300)
    assert ((o - ro).abs() <= bo).all(), f"o: {over.max().item():.2f} of its bound"
    fin = torch.isfinite(rl)
    dl = (lse[fin] - rl[fin]).abs()
    assert (dl <= bl[fin]).all(), f"lse: {(dl / bl[fin]).max().item():.2f} of its bound"


def rotate(x, pos, inv_freq, interleaved):
    """x [..., n, 128] turned to positions pos [n], in 64 bits."""
    x = x.double().clone()
    r = 2 * len(inv_freq)
    angle = pos.double()[:, None] * inv_freq.double().cpu()
    c, s = angle.cos(), angle.sin()
    i0 = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    i1 = i0 + 1 if interleaved else i0 + r // 2
    a, b = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = a * c - b * s, b * c + a * s
    return x
