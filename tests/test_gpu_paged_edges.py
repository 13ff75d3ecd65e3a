"""Edges of the paged-cache calls: sequences that take no part in a call, limits of the arguments, layouts
that differ only where a dimension has one entry, and what a call leaves behind.  Bounds as in
paged_reference.py; every cache has NaN in all slots that hold no token."""
import ctypes

import pytest
import torch

import usagi_b200 as ub
from usagi_b200 import _lib
from paged_reference import Cache, attention, check_attention
from test_paged_args import Call

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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _expect_page_error():
    with pytest.raises(ub.BsattnError) as err:
        ub.check_errors(DEV)
    assert err.value.code == _lib.E_PAGE
    ub.check_errors(DEV)  # cleared


# (prefix, B, Hq, Tq, width): one row and a few by the few-row kernel, up to 32 sequences and more, several
# tiles of rows; many rows; behind a prefix that is read once.
IDLE = {"one_row": (0, 3, 4, 1, 1), "rows": (0, 4, 4, 3, 1), "sequences": (0, 40, 4, 1, 1),
        "row_tiles": (0, 3, 8, 6, 1), "many_rows": (0, 3, 8, 40, 1), "wide": (0, 4, 8, 9, 2200),
        "prefix": (2048, 66, 4, 1, 1), "prefix_rows": (2048, 70, 4, 5, 1)}


@pytest.mark.parametrize("entry", ["none", "recycled"])
@pytest.mark.parametrize("name,window,glob", [(n, w, g) for n in IDLE for w, g in (
    [(None, 0)] if IDLE[n][0] else [(None, 0), (2, 0), (1, 1)])])
def test_a_sequence_without_live_rows_is_not_read(name, window, glob, entry):
    """q_lens[b] == 0: none of its pages is needed, so their entries may be no page at all or pages that
    hold something else by now; its rows are padding."""
    prefix, B, Hq, Tq, width = IDLE[name]
    lens = [prefix + [700, 300, 1283, 129][b % 4] for b in range(B)]
    c = Cache(lens, 2, 16, F16, 211, DEV, prefix=prefix, width_extra=width)
    q, q_lens = _q(B, Hq, Tq, F16, 212), [0 if b % 3 == 1 else Tq for b in range(B)]
    kp, vp, table, sl = c.to(DEV)
    free = next(i for i in range(kp.shape[0]) if torch.isnan(kp[i]).all())
    for b in range(1, B, 3):
        table[b, prefix // 16:] = -1 if entry == "none" else free
    kw = dict(prefix_len=prefix) if prefix else dict(window=window, global_blocks=glob)
    fn = ub.shared_prefix_attn_fwd if prefix else ub.paged_attn_fwd
    o, lse = fn(q.to(DEV), kp, vp, table, sl, q_lens=_ints(q_lens), **kw)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, q_lens, window or 0, glob))


@pytest.mark.parametrize("Tq,Hq", [(1, 8), (5, 4), (200, 2)])
@pytest.mark.parametrize("glob", [1 << 24, (1 << 24) - 1, 1 << 20])
def test_global_blocks_up_to_the_limit(glob, Tq, Hq):
    """More global blocks than a sequence has: every key up to the row's own."""
    c = Cache([700, 2000, 130], 2, 32, F16, 221, DEV)
    q = _q(3, Hq, Tq, F16, 222)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV), window=1, global_blocks=glob)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c, None, 1, glob))


def _odd_strides(x):
    """x with strides of no use (1, 3, 5) in its dimensions of one entry."""
    s = [o if n == 1 else st for n, st, o in zip(x.shape, x.stride(), (3, 5, 1, 1))]
    return torch.as_strided(x, x.shape, s)


@pytest.mark.parametrize("B,H,Tq", [(3, 2, 1), (1, 2, 3), (2, 1, 2), (1, 1, 1)])
def test_strides_of_dimensions_of_one_entry_do_not_matter(B, H, Tq):
    c = Cache([40, 33, 20][:B], H, 16, F16, 231, DEV)
    q, k, v = [_q(B, H, Tq, F16, 232 + i).to(DEV) for i in range(3)]
    inv = ub.rope_inv_freq(128, device=DEV)
    a, b = c.to(DEV), c.to(DEV)
    want = ub.paged_kv_append(*a, k, v, q=q, inv_freq=inv)
    got = ub.paged_kv_append(*b, _odd_strides(k), _odd_strides(v), q=_odd_strides(q), inv_freq=inv)
    assert torch.equal(got, want)
    for x, y in zip(a[:2], b[:2]):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    o, lse = ub.paged_attn_fwd(want, *a)
    o2, lse2 = ub.paged_attn_fwd(_odd_strides(want), *b)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    # a token made by a transpose: its stride over the one token is 1
    one = torch.randn(B, H, 128, 1, generator=torch.Generator().manual_seed(235)).half().to(DEV)
    got = ub.paged_kv_append(*b, one.transpose(2, 3), one.transpose(2, 3))
    assert got is None
    ub.check_errors(DEV)


@pytest.mark.parametrize("Tq,Hq", [(1, 4), (40, 16)])
def test_strides_of_one_page_or_head_do_not_matter(Tq, Hq):
    c = Cache([900], 1, 1024, F16, 236, DEV, extra_pages=0, width_extra=0)
    q = _q(1, Hq, Tq, F16, 237).to(DEV)
    kp, vp, table, lens = c.to(DEV)
    kp, vp = _odd_strides(kp), _odd_strides(vp)
    assert kp.stride() == (3, 5, 128, 1)
    x = c.pages[0][c.table[0, 0].long(), :, 900 - Tq:900][None].to(DEV)
    y = c.pages[1][c.table[0, 0].long(), :, 900 - Tq:900][None].to(DEV)
    ub.paged_kv_append(kp, vp, table, lens, x, y)
    o, lse = ub.paged_attn_fwd(q, kp, vp, table, lens)
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q.cpu(), c))


def test_unsigned_64_bit_metadata():
    """As for signed: what 32 bits do not hold stays out of range, what they hold is taken."""
    c = Cache([40, 33], 2, 16, F16, 241, DEV)
    (kp, vp, table, lens), q = c.to(DEV), _q(2, 4, 1, F16, 242)
    table = table.clamp(min=0)  # the entries behind the sequences
    wide = lambda x, far=0: (x.cpu().long() + far).to(torch.uint64).to(DEV)  # noqa: E731
    top = lambda x: (x.cpu().long() - 2 ** 63).to(torch.uint64).to(DEV)  # noqa: E731
    o, lse = ub.paged_attn_fwd(q.to(DEV), kp, vp, wide(table), wide(lens),
                               q_lens=wide(torch.ones(2)))
    ub.check_errors(DEV)
    check_attention(o, lse, attention(q, c))
    for bad in (dict(block_table=wide(table, 2 ** 32)), dict(seq_lens=wide(lens, 2 ** 32)),
                dict(q_lens=wide(torch.ones(2), 2 ** 32)), dict(block_table=top(table)),
                dict(seq_lens=top(lens)), dict(q_lens=top(torch.ones(2)))):
        kw = dict(block_table=table, seq_lens=lens, q_lens=None)
        kw.update(bad)
        ub.paged_attn_fwd(q.to(DEV), kp, vp, **kw)
        _expect_page_error()


@pytest.mark.parametrize("Tq", [1, 3])
def test_append_writes_nothing_for_a_length_or_count_out_of_range(Tq):
    """A sequence that has outgrown its table row, or a count of rows that the call does not have: there is no
    right slot for its tokens, so the ones that are held stay, and its rows of q are zero."""
    c = Cache([64, 40, 30], 2, 16, F16, 251, DEV, width_extra=0)
    kp, vp, table, lens = c.to(DEV)
    table = torch.where(table < 0, table.flatten()[0], table)  # a page behind a sequence, if one were used
    inv = ub.rope_inv_freq(128, device=DEV)
    k, v = _q(3, 2, Tq, F16, 252).to(DEV), _q(3, 2, Tq, F16, 253).to(DEV)
    q = _q(3, 4, Tq, F16, 254).to(DEV)
    same = torch.full((3,), Tq, dtype=torch.int32, device=DEV)
    good = [x.clone() for x in (kp, vp)]
    want_q = ub.paged_kv_append(*good, table, lens, k, v, q=q, inv_freq=inv)
    ub.check_errors(DEV)
    want_q[0] = 0
    slots = [(table[0, (64 - Tq + t) // 16].item(), (64 - Tq + t) % 16) for t in range(Tq)]
    for x, y in zip(good, (kp, vp)):
        for page, slot in slots:
            x[page, :, slot] = y[page, :, slot]
    for which, value in [("len", 65), ("len", -1), ("len", 2 ** 31 - 1), ("rows", Tq + 1), ("rows", -1),
                         ("rows", 2 ** 31 - 1)]:
        bad = [lens.clone(), same.clone()]
        bad[which == "rows"][0] = value
        a = [x.clone() for x in (kp, vp)]
        got = ub.paged_kv_append(*a, table, bad[0], k, v, q=q, q_lens=bad[1], inv_freq=inv)
        _expect_page_error()
        assert torch.equal(got, want_q), (which, value)
        for x, y in zip(a, good):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16)), (which, value)


def test_a_call_of_much_scratch_keeps_none():
    """Its scratch goes back when it ends, and the stream keeps no other in its place."""
    B, prefix = 1024, 512
    c = Cache([prefix + 1] * B, 8, 64, F16, 261, DEV, prefix=prefix, extra_pages=0, width_extra=0)
    q, args = _q(B, 8, 1, F16, 262), c.to(DEV)
    qd = q.to(DEV)
    stream = torch.cuda.Stream(DEV, priority=-1)
    stream.wait_stream(torch.cuda.current_stream(DEV))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(DEV)
    with torch.cuda.stream(stream):
        torch.cuda.reset_peak_memory_stats(DEV)
        o, lse = ub.shared_prefix_attn_fwd(qd, *args, prefix_len=prefix)
        ub.check_errors(DEV)
    assert torch.cuda.max_memory_allocated(DEV) - before > 32 << 20  # it needs more than is ever kept
    kept = torch.cuda.memory_allocated(DEV) - before - o.nbytes - lse.nbytes
    assert kept < 1 << 20, kept
    check_attention(o[:8], lse[:8], [x[:8] for x in attention(q[:8], c)])


def test_scratch_is_kept_for_a_few_streams_only():
    """A call of 20 MB of scratch on 32 streams: those that were used last keep theirs."""
    c = Cache([900, 400], 2, 64, F16, 271, DEV, width_extra=100)
    q, args = _q(2, 8, 40, F16, 272).to(DEV), c.to(DEV)
    want = ub.paged_attn_fwd(q, *args)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(DEV)
    streams = [torch.cuda.Stream(DEV, priority=-1) for _ in range(32)]
    assert len({s.cuda_stream for s in streams}) > 24
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                o, lse = ub.paged_attn_fwd(q, *args)
                ub.check_errors(DEV)
                assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    del o, lse
    assert torch.cuda.memory_allocated(DEV) - before <= 16 * (33 << 20)


def test_a_call_past_the_limits_says_so():
    """What the C ABI refuses reaches the user with a text that is about these calls."""
    pages = torch.zeros(1, 32, 1024, 128, dtype=F16, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(256, 2048)
    lens = torch.ones(256, dtype=torch.int32, device=DEV)
    q = torch.zeros(256, 32, 1, 128, dtype=F16, device=DEV)
    for kw in (dict(block_table=table), dict(block_table=table[:, :64], window=(1 << 24) + 1)):
        with pytest.raises(ub.BsattnError, match="paged") as err:
            ub.paged_attn_fwd(q, pages, pages, seq_lens=lens, **kw)
        assert err.value.code == _lib.E_SHAPE and "limits" in str(err.value)
    o, lse = ub.paged_attn_fwd(q, pages, pages, table[:, :64], lens)
    ub.check_errors(DEV)
    assert (o == 0).all() and (lse == 0).all()


@pytest.mark.parametrize("Tq", [1, 32])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,mag", [(F16, 200.0), (F16, 30000.0), (BF16, 1e10), (BF16, 1e17)])
def test_scores_of_any_size(dtype, mag, sign, Tq):
    """One product per score, so that 32 bits hold it to half a step; the largest score is at least 2^-8 of its
    size ahead of the others, whose weights vanish.  o is the value of that key, lse its score."""
    n, H, G = 700, 1, 8
    c = Cache([n], H, 32, dtype, 281, DEV)
    g = torch.Generator().manual_seed(282)
    x = sign * mag * (1 + torch.randperm(64, generator=g) / 64.0)
    x = torch.cat([x, torch.full((n - 64,), mag * (0.5 if sign > 0 else -2.1))])
    for j in range(n):
        c.pages[0][c.table[0, j // 32], :, j % 32] = 0
        c.pages[0][c.table[0, j // 32], 0, j % 32, 5] = x[j].to(dtype)
    q = torch.zeros(1, G, Tq, 128, dtype=dtype)
    q[..., 5] = (mag * (1 + torch.rand(1, G, Tq, generator=g))).to(dtype)
    o, lse = ub.paged_attn_fwd(q.to(DEV), *c.to(DEV))
    ub.check_errors(DEV)
    s = c.dense(0, n, 0)[0, :, 5]
    top = int(s.argmax())
    v = c.dense(0, n, 1)[0, top]
    u = torch.finfo(dtype).eps / 2
    assert ((o.double().cpu() - v).abs() <= 2 * u * v.abs()).all()
    want = q[..., 5].double() * s[top] * 128 ** -0.5
    # score, scale_log2, their product, times ln 2: half a step each, and the constants' own
    assert ((lse.double().cpu() - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()


def test_counts_left_behind_do_not_stay():
    """What a call that went wrong leaves in the counters (its lengths were rewritten while it ran, say) is
    gone for the call after the next one of the same buffer, whatever other buffers are used between."""
    c = Cache([20011, 3000], 1, 64, F16, 291, DEV)
    q = _q(2, 2, 1, F16, 292).to(DEV)
    args = c.to(DEV)
    want, want_lse = ub.paged_attn_fwd(q, *args)
    ub.check_errors(DEV)
    kp, vp, table, lens = args
    lib = _lib.load()
    need = ctypes.c_size_t()
    assert lib.bsattn_paged_scratch_bytes(2, 2, 1, 1, table.shape[1], 64, 0, ctypes.byref(need)) == 0
    scratch = torch.empty(need.value, dtype=torch.uint8, device=DEV)
    counters = torch.ones(lib.bsattn_paged_counters(), dtype=torch.int32, device=DEV)
    ws = torch.zeros(lib.bsattn_workspace_bytes() // 4 + 1, dtype=torch.int32, device=DEV)
    call = Call(kp.data_ptr(), vp.data_ptr(), (ctypes.c_int64 * 6)(*kp.stride()[:3], *vp.stride()[:3]),
                table.data_ptr(), table.stride(0), lens.data_ptr(), None, table.shape[1], kp.shape[0], 64,
                2, 2, 1, 1, _lib.OUT_F16, ws.data_ptr(), ws.numel() * 4,
                torch.cuda.current_stream(DEV).cuda_stream)
    for i in range(5):
        ub.paged_attn_fwd(q, *args)
        o, lse = torch.full_like(want, float("nan")), torch.full_like(want_lse, float("nan"))
        assert lib.bsattn_paged_fwd(ctypes.byref(call), q.data_ptr(), o.data_ptr(), lse.data_ptr(), 0, 0, 0,
                                    0.0, scratch.data_ptr(), need.value, counters.data_ptr()) == 0
        torch.cuda.synchronize()
        if i > 0:
            assert torch.equal(o, want) and torch.equal(lse, want_lse), i
    assert (counters == 0).all() and (ws == 0).all()
