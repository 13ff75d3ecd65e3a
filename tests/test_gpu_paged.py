"""Paged-cache operators on the GPU against the 64-bit restatement in paged_reference.py, whose
bounds are derived there.  Every cache has NaN in all slots that hold no token and table entries out
of range behind each sequence, so anything read from there shows."""
import pytest
import torch

import usagi_b200 as ub
from usagi_b200 import _lib
from paged_reference import Cache, attention, check_attention, rotate

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _setup():
    ub.setup(device="cuda:0")
    yield
    ub.check_errors(DEV)


def _q(B, Hq, Tq, dtype, seed, gain=2.0):
    return (gain * torch.randn(B, Hq, Tq, 128,
                               generator=torch.Generator().manual_seed(seed))).to(dtype)


def _ql(q_lens):
    return None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device=DEV)


# (lens, Hq, Hkv, Tq, q_lens, page, dtype, layout)
DECODE = {
    "one_token": ([1], 4, 4, 1, None, 16, F16, "hnd"),
    "empty_and_short": ([0, 1, 2, 15, 16, 17, 127, 128, 129], 8, 2, 1, None, 16, BF16, "hnd"),
    "odd_group": ([333, 40, 700], 6, 2, 1, None, 32, F16, "nhd"),
    "group7": ([513, 255], 28, 4, 1, None, 64, BF16, "hnd"),
    "group16": ([1000, 1], 32, 2, 1, None, 128, F16, "hnd"),
    "group9_over_eight_rows": ([600], 9, 1, 1, None, 256, BF16, "nhd"),
    "long_split": ([20011], 2, 1, 1, None, 64, F16, "hnd"),
    "many_sequences": (list(range(0, 600, 2)), 2, 1, 1, None, 16, F16, "hnd"),
    "page1024": ([3000, 1024], 4, 2, 1, None, 1024, BF16, "hnd"),
    "drafts": ([5, 300, 4099], 8, 4, 5, None, 32, F16, "hnd"),
    "drafts_ragged": ([700, 300, 40, 9], 14, 2, 4, [4, 0, 3, 1], 16, BF16, "nhd"),
    "more_rows_than_tokens": ([3, 0], 4, 2, 6, None, 16, F16, "hnd"),
    "group32_rows": ([300, 77], 32, 1, 1, None, 16, BF16, "hnd"),
    "chunk": ([900, 130], 4, 2, 130, [130, 77], 64, F16, "hnd"),
    "chunk_odd": ([700, 333], 6, 2, 100, [100, 99], 32, BF16, "nhd"),
    "chunk_group5": ([513], 5, 1, 257, None, 128, F16, "hnd"),
    "rows17": ([200, 1111], 17, 1, 1, None, 16, F16, "hnd"),
    "group_over_128_rows_per_token": ([300], 130, 1, 1, None, 64, BF16, "hnd"),
}


@pytest.mark.parametrize("name", list(DECODE))
def test_attention_over_the_cache(name):
    lens, Hq, Hkv, Tq, q_lens, page, dtype, layout = DECODE[name]
    c = Cache(lens, Hkv, page, dtype, 11, DEV, layout)
    q = _q(len(lens), Hq, Tq, dtype, 12)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV), q_lens=_ql(q_lens))
    ub.check_errors(DEV)
    assert o.dtype == dtype and o.shape == q.shape
    check_attention(o, lse, attention(q, c, q_lens))


@pytest.mark.parametrize("name", ["odd_group", "group9_over_eight_rows", "group16", "drafts",
                                  "drafts_ragged", "more_rows_than_tokens", "group32_rows", "chunk_odd",
                                  "rows17"])
def test_in_a_wide_table(name):
    """What a call may hold decides the kernel for more than 8 rows a head; the table's unused width
    counts for that and changes nothing else."""
    lens, Hq, Hkv, Tq, q_lens, page, dtype, layout = DECODE[name]
    c = Cache(lens, Hkv, page, dtype, 11, DEV, layout, width_extra=70016 // page)
    q = _q(len(lens), Hq, Tq, dtype, 12)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV), q_lens=_ql(q_lens))
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, q_lens))


@pytest.mark.parametrize("Hq,Hkv,Tq,B", [(32, 8, 4, 4), (4, 1, 32, 3), (14, 2, 9, 2), (16, 16, 64, 1),
                                         (128, 1, 1, 1), (5, 5, 27, 7)])
@pytest.mark.parametrize("window,glob", [(None, 0), (1, 1)])
def test_small_calls_of_many_rows(Hq, Hkv, Tq, B, window, glob):
    c = Cache(_cycle([333, 90, 5, 256], B), Hkv, 16, BF16, 13, DEV)
    q = _q(B, Hq, Tq, BF16, 14)
    q_lens = _cycle([Tq, max(Tq - 3, 0), 1], B)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV), q_lens=_ql(q_lens), window=window,
                               global_blocks=glob)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, q_lens, window or 0, glob))


@pytest.mark.parametrize("Tq", [1, 5, 40, 200])
def test_pages_outside_the_window_need_not_exist(Tq):
    """Pages wholly outside the blocks that any row sees are not read: their entries may be anything."""
    lens, page, window, glob = [1000, 1283, 700], 64, 2, 1
    c = Cache(lens, 2, page, F16, 23, DEV)
    q = _q(3, 4, Tq, F16, 24)
    kp, vp, table, sl = c.to(DEV)
    for b, n in enumerate(lens):
        lo = (max(n - Tq, 0) // 128 - window + 1) * 128
        table[b, glob * 128 // page:max(lo, 0) // page] = -1
    assert (table[:, 2:6] == -1).any()
    o, lse = ub.paged_attn_fwd(q.to(DEV), kp, vp, table, sl, window=window, global_blocks=glob)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, None, window, glob))


@pytest.mark.parametrize("window,glob", [(1, 0), (2, 1), (3, 4), (64, 2)])
@pytest.mark.parametrize("Tq,Hq", [(1, 8), (5, 4), (200, 2)])
def test_window_and_global_blocks(window, glob, Tq, Hq):
    lens = [200, 640, 1283, 2000]
    c = Cache(lens, 2, 32, F16, 21, DEV)
    q = _q(4, Hq, Tq, F16, 22)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV), window=window, global_blocks=glob)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, None, window, glob))


def _cycle(values, n):
    return [values[i % len(values)] for i in range(n)]


# (prefix, own lens, Hq, Hkv, Tq, q_lens, page, dtype, layout).  A prefix is read once when that saves
# 128 MB (512 bytes a token and head for every sequence but one); the first seven save less.
SHARED = {
    "small": (64, [1, 7, 30], 8, 2, 1, None, 16, F16, "hnd"),
    "no_prefix": (0, [100, 40], 4, 2, 1, None, 32, BF16, "hnd"),
    "drafts": (320, [5, 6, 70, 9, 33], 8, 2, 5, [5, 2, 0, 4, 5], 64, F16, "nhd"),
    "chunks": (256, [70, 200], 4, 2, 70, [70, 33], 32, BF16, "hnd"),
    "long_chunks": (256, [300], 2, 1, 300, None, 64, F16, "hnd"),
    "one_sequence": (1280, [1], 4, 4, 1, None, 64, F16, "hnd"),
    "shorter_than_the_prefix": (256, [-256, -100, -1, 0, 1, 40], 8, 2, 1, None, 64, F16, "hnd"),
    "once_ends_inside_a_tile": (2064, _cycle([1, 200, 129], 130), 8, 1, 1, None, 16, BF16, "nhd"),
    "once_whole_tiles": (2048, [3] * 67, 16, 2, 1, None, 128, F16, "hnd"),
    "once_odd_group": (2096, list(range(1, 67)), 6, 2, 1, None, 16, F16, "hnd"),
    "once_group7": (2064, list(range(1, 131)), 7, 1, 1, None, 16, BF16, "hnd"),
    "once_group16": (2080, _cycle([1, 140, 33], 130), 16, 1, 1, None, 32, F16, "nhd"),
    "once_equal_heads": (1040, _cycle([5, 60], 66), 4, 4, 1, None, 16, BF16, "hnd"),
    "once_drafts": (2112, _cycle([5, 6, 70, 9, 33], 130), 4, 1, 5, _cycle([5, 2, 0, 4, 5], 130), 64,
                    F16, "nhd"),
    "once_rows33": (2064, _cycle([11, 40], 130), 3, 1, 11, _cycle([11, 3], 130), 16, BF16, "hnd"),
    "once_rows64": (2048, [70] * 130, 4, 1, 16, None, 256, F16, "hnd"),
    "once_shorter": (4096, _cycle([-4096, -3000, -1, 0, 1, 40, -90], 66), 4, 1, 1, None, 64, F16,
                     "hnd"),
    "once_rows_end_inside": (4096, _cycle([-100, 3, 2, -1, -4090], 66), 4, 1, 8,
                             _cycle([8, 8, 1, 0, 8], 66), 64, BF16, "hnd"),
    "once_few_long_rows": (32768, [40, 1, 7], 8, 4, 1, None, 64, F16, "hnd"),
}


@pytest.mark.parametrize("name", list(SHARED))
def test_shared_prefix(name):
    prefix, own, Hq, Hkv, Tq, q_lens, page, dtype, layout = SHARED[name]
    lens = [prefix + n for n in own]
    c = Cache(lens + [prefix], Hkv, page, dtype, 31, DEV, layout, prefix=prefix)
    c.table, c.lens = c.table[:-1], c.lens[:-1]  # the last one only holds the whole prefix
    q = _q(len(lens), Hq, Tq, dtype, 32)
    o, lse = ub.shared_prefix_attn_fwd(q.to(DEV), *c.to(DEV), prefix_len=prefix,
                                       q_lens=_ql(q_lens))
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, q_lens))


def test_scores_far_apart():
    """Key blocks of growing size raise the running maximum again and again; a huge score makes
    every other weight vanish."""
    c = Cache([1500, 700], 2, 32, F16, 41, DEV)
    k = c.pages[0]
    for b, n in enumerate(c.lens):
        for j in range(n):
            k[c.table[b, j // 32], :, j % 32] *= 0.2 + j / 150
    q = _q(2, 8, 1, F16, 42, gain=4.0)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV))
    check_attention(o, lse, attention(q, c))
    # more rows on the same keys
    q = _q(2, 8, 7, F16, 43, gain=4.0)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV))
    check_attention(o, lse, attention(q, c))
    # and one of the sequences as a prefix that 130 rows share
    args = [x[:1].expand(130, *x.shape[1:]) if i > 1 else x for i, x in enumerate(c.to(DEV))]
    q = _q(130, 8, 1, F16, 44, gain=4.0)
    o, lse = ub.shared_prefix_attn_fwd(q.to(DEV), *args, prefix_len=1024)
    c.table, c.lens = c.table[:1].expand(130, -1), [c.lens[0]] * 130
    check_attention(o, lse, attention(q, c))
    ub.check_errors(DEV)


@pytest.mark.parametrize("prefix,B,Tq", [(0, 2, 1), (0, 2, 3), (256, 2, 3), (2048, 66, 2)])
def test_options(prefix, B, Tq):
    """Scale, output type, given outputs, no lse, int64 metadata, a strided table and q."""
    c = Cache(_cycle([prefix + 44, prefix + 244], B), 2, 64, BF16, 51, DEV, prefix=prefix)
    q = _q(B, 4, Tq, BF16, 52)
    kp, vp, table, lens = c.to(DEV)
    kw = dict(prefix_len=prefix) if prefix else {}
    fn = ub.shared_prefix_attn_fwd if prefix else ub.paged_attn_fwd
    qs = q.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    wide = torch.full((B, 2 * table.shape[1]), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    out = torch.empty(B, 4, Tq, 128, device=DEV, dtype=F16)
    lse = torch.empty(B, 4, Tq, device=DEV)
    o, l2 = fn(qs, kp, vp, wide[:, :table.shape[1]], lens.long(), scale=0.05, out_dtype=F16,
               out=out, lse_out=lse, **kw)
    assert o is out and l2 is lse
    check_attention(o, lse, attention(q, c, scale=0.05, out_dtype=F16))
    o, none = fn(q.to(DEV), kp, vp, table, lens, return_lse=False, **kw)
    assert none is None
    want = attention(q, c)
    check_attention(o, want[1], want)
    ub.check_errors(DEV)


APPEND = {
    # lens, q_lens, Hq, Hkv, Tq, page, dtype, layout, rot, interleaved
    "one": ([1], None, 4, 4, 1, 16, F16, "hnd", 128, False),
    "batch": ([17, 1, 33, 500, 64], None, 8, 2, 1, 16, BF16, "nhd", 128, False),
    "ragged_interleaved": ([40, 7, 300], [5, 0, 3], 6, 3, 5, 32, F16, "hnd", 64, True),
    "prompt": ([130, 129], [130, 100], 2, 1, 130, 64, BF16, "hnd", 32, False),
    "no_rotation": ([20, 19], None, 4, 2, 3, 16, F16, "nhd", 0, False),
    "odd_rot": ([1000, 999], None, 3, 3, 2, 256, F16, "hnd", 48, False),
    "full_interleaved": ([1000, 64], None, 3, 1, 2, 1024, BF16, "hnd", 128, True),
    "no_q": ([90, 3], [2, 3], 0, 2, 3, 16, BF16, "hnd", 128, False),
}


@pytest.mark.parametrize("name", list(APPEND))
def test_append(name):
    lens, q_lens, Hq, Hkv, Tq, page, dtype, layout, rot, inter = APPEND[name]
    c = Cache(lens, Hkv, page, dtype, 61, DEV, layout)
    B = len(lens)
    g = torch.Generator().manual_seed(62)
    qkv = torch.randn(B, Tq, Hq + 2 * Hkv, 128, generator=g).to(dtype)
    dev = qkv.to(DEV)
    q, k, v = [x.transpose(1, 2) for x in dev.split([Hq, Hkv, Hkv], 2)]
    inv = ub.rope_inv_freq(rot, 10000.0, DEV) if rot else None
    kp, vp, table, sl = c.to(DEV)
    out = ub.paged_kv_append(kp, vp, table, sl, k, v, q=q if Hq else None, q_lens=_ql(q_lens),
                             inv_freq=inv, interleaved=inter)
    ub.check_errors(DEV)
    u = torch.finfo(dtype).eps / 2
    want_k, want_v = [x.clone() for x in c.pages]
    close = torch.zeros_like(want_k, dtype=torch.bool)
    hq, hk, hv = [x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], 2)]

    def near(got, exact, pair):
        """One rounding, after 32-bit products of values no larger than the pair's length."""
        return (got.double().cpu() - exact).abs() <= u * exact.abs() + 2.0 ** -21 * pair + 2.0 ** -25

    for b, L in enumerate(lens):
        n = Tq if q_lens is None else q_lens[b]
        pos = torch.arange(L - n, L)
        turn = (lambda x: rotate(x, pos, inv.cpu(), inter)) if rot else (lambda x: x.double())
        big = (lambda x: x.double().abs().amax(-1, keepdim=True)) if rot else (lambda x: 0.0)
        if Hq:
            assert near(out[b, :, :n], turn(hq[b, :, :n]), big(hq[b, :, :n])).all()
            assert (out[b, :, n:] == 0).all()
        page_of, slot = c.table[b, pos // page].long(), pos % page
        got = kp.cpu()[page_of, :, slot].transpose(0, 1)
        assert near(got, turn(hk[b, :, :n]), big(hk[b, :, :n])).all()
        want_k[page_of, :, slot] = got.transpose(0, 1)
        want_v[page_of, :, slot] = hv[b, :, :n].transpose(0, 1)
    if not Hq:
        assert out is None
    # every other slot, and all of v, bit for bit
    for got, want in ((kp, want_k), (vp, want_v)):
        assert torch.equal(got.cpu().contiguous().view(torch.int16),
                           want.contiguous().view(torch.int16))


def test_append_far_positions():
    """At position two million the angle has to be formed in 64 bits."""
    page, n = 1024, 2_000_003
    table = torch.full((1, n // page + 1), 0, dtype=torch.int32, device=DEV)
    kp, vp = [torch.zeros(1, 1, page, 128, dtype=F16, device=DEV) for _ in range(2)]
    x = torch.randn(1, 1, 1, 128, generator=torch.Generator().manual_seed(63)).half()
    inv = ub.rope_inv_freq(128, 500000.0, DEV)
    q = ub.paged_kv_append(kp, vp, table, torch.tensor([n], device=DEV), x.to(DEV), x.to(DEV),
                           q=x.to(DEV), inv_freq=inv)
    want = rotate(x, torch.tensor([n - 1]), inv, False)
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -20 * x.double().abs().max()
    assert ((q.double().cpu() - want).abs() <= bound).all()
    ub.check_errors(DEV)


def test_append_in_place_and_unaligned():
    c = Cache([100, 30], 2, 16, BF16, 71, DEV)
    g = torch.Generator().manual_seed(72)
    q, k, v = [torch.randn(2, h, 4, 128, generator=g).to(BF16).to(DEV) for h in (4, 2, 2)]
    inv = ub.rope_inv_freq(128, device=DEV)
    a, b = c.to(DEV), c.to(DEV)
    want = ub.paged_kv_append(*a, k, v, q=q, inv_freq=inv)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    same = q.clone()
    got = ub.paged_kv_append(*b, k, v, q=same, inv_freq=inv, q_out=same)
    assert got is same and torch.equal(got, want)
    assert torch.equal(ub.paged_kv_append(*b, k, v, q=odd, inv_freq=inv), want)
    for x, y in zip(a[:2], b[:2]):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    ub.check_errors(DEV)


def _expect_page_error():
    with pytest.raises(ub.BsattnError) as err:
        ub.check_errors(DEV)
    assert err.value.code == _lib.E_PAGE
    ub.check_errors(DEV)  # cleared


@pytest.mark.parametrize("prefix,B,Tq,width", [(0, 3, 1, 1), (0, 3, 40, 1), (0, 3, 40, 2200),
                                               (128, 3, 1, 1), (2048, 66, 3, 1)])
def test_bad_pages_and_lengths_are_reported(prefix, B, Tq, width):
    """Out-of-range table entries, lengths and row counts are found and reported; the sequences
    that are in order keep their results."""
    lens_ = _cycle([prefix + 200, prefix + 190, prefix + 180], B)
    c = Cache(lens_, 2, 16, F16, 81, DEV, prefix=prefix, width_extra=width)
    q = _q(B, 4, Tq, F16, 82).to(DEV)
    kp, vp, table, lens = c.to(DEV)
    fn = (lambda *a, **k: ub.shared_prefix_attn_fwd(*a, prefix_len=prefix, **k)) if prefix \
        else ub.paged_attn_fwd
    ref = fn(q, kp, vp, table, lens)
    ub.check_errors(DEV)
    want = attention(q.cpu(), c)
    others = [b for b in range(B) if b != 1]

    def in_order(o, lse, which):
        check_attention(o[which], lse[which], [x[which] for x in want])

    in_order(*ref, list(range(B)))
    for value in (-1, kp.shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[1, prefix // 16 + 9] = value
        o, lse = fn(q, kp, vp, bad, lens)
        _expect_page_error()
        for b in others:
            assert torch.equal(o[b], ref[0][b]) and torch.equal(lse[b], ref[1][b])
    for value in (-5, table.shape[1] * 16 + 1, 2 ** 31 - 1):
        bad = lens.clone()
        bad[1] = value
        # the pages a longer length reaches exist in the table's width only
        ok = table.clamp(min=0)
        o, lse = fn(q, kp.nan_to_num(), vp.nan_to_num(), ok, bad)
        _expect_page_error()
        in_order(o, lse, others)
    for value in (-1, Tq + 1, 2 ** 31 - 1):
        ql = torch.full((B,), Tq, dtype=torch.int32, device=DEV)
        ql[1] = value
        o, lse = fn(q, kp, vp, table, lens, q_lens=ql)
        _expect_page_error()
        in_order(o, lse, others)
    if prefix:
        bad = table.clone()
        bad[0, 5] = kp.shape[0]
        fn(q, kp, vp, bad, lens)
        _expect_page_error()


def test_refusals():
    """What the calls refuse before a launch, with the exception it raises."""
    c = Cache([40, 33], 2, 16, F16, 84, DEV)
    kp, vp, table, lens = c.to(DEV)
    q, k = _q(2, 4, 1, F16, 85).to(DEV), _q(2, 2, 1, F16, 86).to(DEV)
    inv = ub.rope_inv_freq(128, device=DEV)
    attn = lambda q=q, kp=kp, vp=vp, table=table, lens=lens, **kw: \
        ub.paged_attn_fwd(q, kp, vp, table, lens, **kw)  # noqa: E731
    append = lambda k=k, v=k, kp=kp, table=table, lens=lens, **kw: \
        ub.paged_kv_append(kp, vp, table, lens, k, v, **kw)  # noqa: E731
    shared = lambda n: ub.shared_prefix_attn_fwd(q, kp, vp, table, lens, prefix_len=n)  # noqa: E731
    tall = torch.zeros(2, 2, 8, 128, dtype=F16, device=DEV)
    odd = torch.zeros(6, 2, 24, 128, dtype=F16, device=DEV)
    for error, calls in ((ValueError, [
            lambda: attn(q=q[0]), lambda: attn(q=q[:1]), lambda: attn(q=q[:, :3].contiguous()),
            lambda: attn(q=q[..., :64].contiguous()), lambda: attn(kp=kp[:, :1], vp=vp),
            lambda: attn(kp=tall, vp=tall), lambda: attn(kp=odd, vp=odd),
            lambda: attn(kp=kp[..., ::2], vp=vp[..., ::2]), lambda: attn(kp=kp[:0], vp=vp[:0]),
            lambda: attn(table=table[0]), lambda: attn(table=table[:1]), lambda: attn(lens=lens[:1]),
            lambda: attn(q_lens=lens[:1]), lambda: attn(out=q[:1]), lambda: attn(out=q.float()),
            lambda: attn(lse_out=torch.zeros(2, 4, device=DEV)), lambda: attn(window=0),
            lambda: attn(global_blocks=1), lambda: attn(window=2, global_blocks=-1),
            lambda: attn(scale=0.0), lambda: attn(scale=-0.1), lambda: attn(scale=float("nan")),
            lambda: attn(scale=1e39),
            lambda: attn(window=2 ** 40), lambda: shared(24), lambda: shared(-16),
            lambda: shared(16 * (table.shape[1] + 1)), lambda: shared(2 ** 40),
            lambda: append(k=k[0]), lambda: append(k=k[:1]), lambda: append(v=q),
            lambda: append(q=q[:1]), lambda: append(q_out=q), lambda: append(q=q, q_out=k),
            lambda: append(q=q, q_out=torch.zeros(2, 4, 1, 256, dtype=F16, device=DEV)[..., :128]),
            lambda: append(q=q, inv_freq=inv[:4]), lambda: append(q=q, inv_freq=inv[:12]),
            lambda: append(inv_freq=torch.zeros(72, dtype=torch.float64, device=DEV))]),
            (TypeError, [
            lambda: attn(q=q.bfloat16()), lambda: attn(q=q.cpu()), lambda: attn(vp=vp.bfloat16()),
            lambda: attn(kp=kp.float(), vp=vp.float(), q=q.float()),
            lambda: attn(out_dtype=torch.float32), lambda: attn(out_dtype=16), lambda: attn(q=None),
            lambda: attn(scale="1"), lambda: append(v=k.bfloat16()), lambda: append(q=q.bfloat16()),
            lambda: append(k=k.cpu()), lambda: append(inv_freq=inv.float()),
            lambda: append(inv_freq=inv.cpu()), lambda: append(inv_freq=inv[None])])):
        for i, call in enumerate(calls):
            with pytest.raises(error):
                call()
                pytest.fail(f"{error.__name__} call {i} was accepted")
    with pytest.raises(ub.BsattnError) as err:  # windows past the C ABI's bound
        attn(window=(1 << 24) + 1)
    assert err.value.code == _lib.E_SHAPE
    # empty batches and no rows are no error
    o, lse = attn(q=q[:0], table=table[:0], lens=lens[:0])
    assert o.shape == (0, 4, 1, 128) and lse.shape == (0, 4, 1)
    o, lse = attn(q=q[:, :, :0])
    assert o.shape == (2, 4, 0, 128)
    assert append(k=k[:, :, :0], v=k[:, :, :0], q=q[:, :, :0]).shape == (2, 4, 0, 128)
    ub.check_errors(DEV)


def test_first_call_on_a_stream_inside_capture_is_refused():
    """As for the prefill calls: the stream's error word has to exist before a capture."""
    from usagi_b200 import api
    c = Cache([40], 2, 16, F16, 87, DEV)
    args, q = c.to(DEV), _q(1, 4, 1, F16, 88).to(DEV)
    fresh = torch.cuda.Stream(DEV)
    fresh.wait_stream(torch.cuda.current_stream(DEV))
    api._workspaces.pop((DEV.index, fresh.cuda_stream), None)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside graph capture"):
        with torch.cuda.graph(graph, stream=fresh):
            ub.paged_attn_fwd(q, *args)
    del graph


def test_wide_integers_and_floats_as_indexes():
    """64-bit metadata whose low 32 bits look right is out of range; floats are refused."""
    c = Cache([40, 33], 2, 16, F16, 87, DEV)
    (kp, vp, table, lens), q = c.to(DEV), _q(2, 4, 1, F16, 88)
    o, lse = ub.paged_attn_fwd(q.to(DEV), kp, vp, table.long(), lens.long(),
                               q_lens=torch.ones(2, dtype=torch.int64, device=DEV))
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c))
    for far in (2 ** 32, -2 ** 32):
        ub.paged_attn_fwd(q.to(DEV), kp, vp, table.long() + far, lens)
        _expect_page_error()
        ub.paged_attn_fwd(q.to(DEV), kp, vp, table, lens.long() + far)
        _expect_page_error()
        ub.paged_attn_fwd(q.to(DEV), kp, vp, table, lens,
                          q_lens=torch.full((2,), 1 + far, dtype=torch.int64, device=DEV))
        _expect_page_error()
    for bad in (dict(block_table=table.float()), dict(seq_lens=lens.half()), dict(q_lens=lens > 0)):
        kw = dict(block_table=table, seq_lens=lens, q_lens=None)
        kw.update(bad)
        with pytest.raises(TypeError, match="integers"):
            ub.paged_attn_fwd(q.to(DEV), kp, vp, **kw)


def test_gradients_are_not_recorded():
    c = Cache([40], 2, 16, F16, 89, DEV)
    args, q = c.to(DEV), _q(1, 4, 1, F16, 90).to(DEV).requires_grad_()
    o, lse = ub.paged_attn_fwd(q, *args)
    assert not o.requires_grad and not lse.requires_grad


def test_append_reports_bad_pages_and_writes_nothing_there():
    c = Cache([40, 40], 1, 16, F16, 83, DEV)
    kp, vp, table, lens = c.to(DEV)
    x = torch.ones(2, 1, 1, 128, dtype=F16, device=DEV)
    before = kp.clone()
    for value in (-1, kp.shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[0, 2] = value
        ub.paged_kv_append(kp, vp, bad, lens, x, x)
        _expect_page_error()
    want = before.clone()
    want[table[1, 2].item(), :, 39 % 16] = 1
    assert torch.equal(kp.view(torch.int16), want.view(torch.int16))
    ub.paged_kv_append(kp, vp, table, torch.tensor([10 ** 6, 40], device=DEV), x, x)
    _expect_page_error()


def _three_calls(seed):
    """A call for each of the ways through the attention kernels, with its arguments."""
    c = Cache([5000 + seed, 3, 777, 1200], 2, 32, BF16, 91 + seed, DEV)
    one, many = _q(4, 8, 1, BF16, 92 + seed).to(DEV), _q(4, 8, 9, BF16, 93 + seed).to(DEV)
    args = c.to(DEV)
    p = Cache(_cycle([2048 + 40 + seed, 2048 + 7], 66), 2, 64, BF16, 94 + seed, DEV, prefix=2048)
    shared, pargs = _q(66, 4, 1, BF16, 95 + seed).to(DEV), p.to(DEV)
    return [lambda: ub.paged_attn_fwd(one, *args), lambda: ub.paged_attn_fwd(many, *args),
            lambda: ub.shared_prefix_attn_fwd(shared, *pargs, prefix_len=2048)]


def test_results_do_not_depend_on_the_run():
    calls = _three_calls(0)
    first = [f() for f in calls]
    for _ in range(5):
        for f, w in zip(calls, first):
            o, lse = f()
            assert torch.equal(o, w[0]) and torch.equal(lse, w[1])
    ub.check_errors(DEV)


def test_two_graphs_side_by_side():
    """Two graphs captured on one stream and replayed at once on two: nothing is shared."""
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    want, outs, graphs = [], [], []
    with torch.cuda.stream(side):
        sets = [_three_calls(s) for s in range(2)]
        for calls in sets:
            want.append([x for f in calls for x in f()])
        side.synchronize()
        for calls in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append([x for f in calls for x in f()])
            graphs.append(graph)
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for rep in range(20):
        for o in outs:
            for x in o:
                x.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        # eager calls of the same sizes between the replays, on a third stream
        eager = [x for f in sets[0] for x in f()]
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(o, w)), rep
        assert all(torch.equal(x, y) for x, y in zip(eager, want[0])), rep
    with torch.cuda.stream(side):
        ub.check_errors(DEV)
    ub.check_errors(DEV)
    del graphs


def test_two_streams_at_once():
    """Calls that overlap on two streams: each stream has its own scratch and counters."""
    sets = [_three_calls(s) for s in range(2)]
    want = [[x for f in calls for x in f()] for calls in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    for rep in range(10):
        outs = [[], []]
        for _ in range(3):
            for s, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    outs[s] = [x for f in sets[s] for x in f()]
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(o, w)), rep
    for stream in streams:
        with torch.cuda.stream(stream):
            ub.check_errors(DEV)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes per tensor whose tokens sit at its end."""
    Hkv, page = 8, 64
    n_pages = (1 << 32) // (Hkv * page * 128 * 2) + 40
    kp, vp = [torch.zeros(n_pages, Hkv, page, 128, dtype=F16, device=DEV) for _ in range(2)]
    L = 20 * page - 5
    c = Cache([L], Hkv, page, F16, 111, DEV, extra_pages=0, width_extra=0)
    first = n_pages - c.pages[0].shape[0]
    kp[first:], vp[first:] = c.pages[0].to(DEV), c.pages[1].to(DEV)
    table = c.table.to(DEV) + first
    lens = torch.tensor([L], dtype=torch.int32, device=DEV)
    q = _q(1, 16, 1, F16, 112)
    want = attention(q, c)
    o, lse = ub.paged_attn_fwd(q.to(DEV), kp, vp, table, lens)
    check_attention(o, lse, want)
    many = _q(1, 16, 9, F16, 114)
    o, lse = ub.paged_attn_fwd(many.to(DEV), kp, vp, table, lens)
    check_attention(o, lse, attention(many, c))
    x = torch.randn(1, Hkv, 1, 128, generator=torch.Generator().manual_seed(113)).half().to(DEV)
    ub.paged_kv_append(kp, vp, table, lens, x, x)
    at = table[0, (L - 1) // page].item(), (L - 1) % page
    assert torch.equal(kp[at[0], :, at[1]], x[0, :, 0])
    assert torch.equal(vp[at[0], :, at[1]], x[0, :, 0])
    ub.check_errors(DEV)


@pytest.mark.parametrize("window,glob", [(None, 0), (2, 1)])
def test_prefill_then_decode(window, glob):
    """The operators together, as a serving loop uses them: a prompt is appended (rotated) and
    prefilled with the framework's window kernel, then tokens are added one by one and attend over
    the cache.  Every step has to agree with the prefill kernel run over the whole sequence."""
    B, H, page, T, steps = 2, 2, 64, 1024, 3
    g = torch.Generator(device=DEV).manual_seed(121)
    q, k, v = [torch.randn(B, H, T, 128, generator=g, device=DEV).half() for _ in range(3)]
    inv = ub.rope_inv_freq(128, 10000.0, DEV)
    kp, vp = [torch.full((B * T // page, H, page, 128), float("nan"), dtype=F16, device=DEV)
              for _ in range(2)]
    table = torch.randperm(B * T // page, generator=torch.Generator().manual_seed(1)).view(B, -1)
    table = table.to(DEV, torch.int32)
    # the whole sequence at once: rotated q, and k read back from the cache
    full = torch.full((B,), T, dtype=torch.int32, device=DEV)
    rq = ub.paged_kv_append(kp, vp, table, full, k, v, q=q, inv_freq=inv)
    rk = kp[table.long()].transpose(1, 2).reshape(B, H, T, 128)
    o_ref, lse_ref = ub.block_sparse_attn_fwd_window(rq, rk, v, window=window or T // 128,
                                                     global_blocks=glob)
    # again: a prompt, then single tokens
    kp.fill_(float("nan"))
    vp.fill_(float("nan"))
    n = T - steps
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    ub.paged_kv_append(kp, vp, table, lens, k[:, :, :n], v[:, :, :n], inv_freq=inv)
    for i in range(n, T):
        lens += 1
        qi = ub.paged_kv_append(kp, vp, table, lens, k[:, :, i:i + 1], v[:, :, i:i + 1],
                                q=q[:, :, i:i + 1], inv_freq=inv)
        assert torch.equal(qi, rq[:, :, i:i + 1])
        o, lse = ub.paged_attn_fwd(qi, kp, vp, table, lens, window=window, global_blocks=glob)
        # both kernels round P and o once each: 2 (u A + u |o|), with A <= max |v|
        bound = 4 * 2.0 ** -11 * v.abs().max().item()
        assert (o - o_ref[:, :, i:i + 1]).abs().max().item() <= bound
        assert (lse - lse_ref[:, :, i:i + 1]).abs().max().item() <= 2e-4
    assert torch.equal(kp[table.long()].transpose(1, 2).reshape(B, H, T, 128), rk)
    ub.check_errors(DEV)


def test_wait_timeout_is_reported_and_context_survives():
    """The many-row kernel's waits are bounded: with the test hook its Q K^T issuers wait on a barrier
    that nothing signals, the bound runs out on every SM, and the host reads the status."""
    calls = _three_calls(0)[1:]
    want = [f() for f in calls]
    ub.check_errors(DEV)
    lib = _lib.load()
    for f, w in zip(calls, want):
        try:
            ub.set_timeout_ns(10_000_000)
            lib.bsattn_test_unsignalled_wait(1)
            f()
            with pytest.raises(ub.BsattnError) as err:
                ub.check_errors(DEV)
            assert err.value.code == _lib.E_TIMEOUT
        finally:
            lib.bsattn_test_unsignalled_wait(0)
            ub.set_timeout_ns(2_000_000_000)
        o, lse = f()
        ub.check_errors(DEV)
        assert torch.equal(o, w[0]) and torch.equal(lse, w[1])
