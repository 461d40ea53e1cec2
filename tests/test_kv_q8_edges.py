"""Attention over the 8-bit paged K/V cache where it can go wrong: precision, the ends of the exponents' range, values that a query
does not see, tables that do not hold what the lengths promise. Oracle in 64 bits: oracle/kv_q8.py."""
import ctypes
import math

import pytest
import torch

from oracle import kv_q8 as ref
from tests.helpers import mean_rel
from tests.test_kv_q8 import _check, _pool, _rows

DEV = "cuda:0"
gpu = pytest.mark.gpu
SCALE = 128 ** -0.5


@pytest.fixture(scope="module")
def ops(sb):
    from spikingbrain_7b_b200 import ops as o
    return o


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(new):
    return _i32(*[sum(new[:i]) for i in range(len(new) + 1)])


def _weights_of(new):
    """What the kernel of these runs holds its weights in."""
    return ref.FP16 if max(new) <= 16 else ref.TWO_BF16


def _attend(ops, q, codes, scales, table, ctx, new, wl, scale=SCALE, status=0, **kw):
    """swa_prefill_q8 (or swa_decode_q8 where `new` is None) on CPU tensors -> output on the GPU, status checked."""
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = [t.to(DEV) for t in (codes[0], codes[1], scales[0], scales[1], table)]
    if new is None:
        out = ops.swa_decode_q8(q.to(DEV), *cache, _i32(*ctx), window_left=wl, scale=scale, status=st, **kw)
    else:
        out = ops.swa_prefill_q8(q.to(DEV), *cache, _starts(new), _i32(*ctx), max(new), window_left=wl, scale=scale, status=st, **kw)
    assert st.item() == status
    return out


# ------------------------------------------------------------------------------------- precision
# The bar of the framework's attention kernels: mean-rel 1e-3 against the definition rounded to the output's type.
MEAN_REL = 1e-3


@gpu
@pytest.mark.parametrize("ctx,new,wl,H,kvh", [([4200], [300], 4096, 28, 4), ([0, 3001], [700, 130], -1, 14, 2),
                                              ([9000], [40], -1, 7, 1), ([500, 70], [17, 64], 300, 4, 4)])
def test_long_runs_hold_their_weights_in_more_bits_than_the_output(ops, ctx, new, wl, H, kvh):
    lens = [a + b for a, b in zip(ctx, new)]
    codes, scales, table = _pool(lens, wl, kvh, 128, 16, seed=200, spread=0.5, n_new=new)
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(201)).bfloat16()
    out = _attend(ops, q, codes, scales, table, ctx, new, wl)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, wl, SCALE, weights=_weights_of(new))
    _check(out, None, want)
    assert mean_rel(out.float(), want[0].bfloat16().float()) <= MEAN_REL


# ------------------------------------------------------------------------------------- the ends of the exponents' range
def _row(codes, scales, table, which, seq, tok, head):
    """The codes [D] of a token's row of K (0) or V (1), and the place of its exponent byte."""
    bs = codes.shape[2]
    blk = int(table[seq, tok // bs])
    return codes.view(torch.uint8)[which, blk, tok % bs, head], (which, blk, head, tok % bs)


@gpu
@pytest.mark.parametrize("new", [None, 2, 3, 4, 16, 40])
@pytest.mark.parametrize("exponent", [57, 58, 63])
@pytest.mark.parametrize("peaked", [False, True])
def test_an_empty_v_row_beside_the_largest_ones(ops, new, exponent, peaked):
    """Token 0 holds zeros (the smallest exponent), the others V rows of the largest. Queries that see token 0 alone, or whose
    softmax leaves nothing for the others, give zeros; the others finite values."""
    H, kvh, n = 28, 4, new or 1
    ctx = [0, 21]
    lens = [2, 22] if new is None else [c + n for c in ctx]
    codes, scales, table = _pool(lens, -1, kvh, 128, 16, seed=210, spread=0.5, n_new=[n, n])
    g = torch.Generator().manual_seed(211)
    u = torch.where(torch.rand(128, generator=g) < 0.5, -1.0, 1.0)
    for s, L in enumerate(lens):
        for h in range(kvh):
            for t in range(L):
                row, at = _row(codes, scales, table, 1, s, t, h)
                if t == 0:
                    row.zero_()
                    key, key_at = _row(codes, scales, table, 0, s, 0, h)
                    key.copy_(u.to(torch.float8_e4m3fn).view(torch.uint8))
                    scales[key_at] = 127
                scales[at] = 63 if t == 0 else 127 + exponent
    q = torch.randn(2 * n, H, 128, generator=g)
    q = ((60.0 * u).expand(2 * n, H, 128) if peaked else q).bfloat16().contiguous()
    out = _attend(ops, q, codes, scales, table, lens if new is None else ctx, None if new is None else [n, n], -1)
    dev = [t.to(DEV) for t in (q, codes, scales, table)]
    want = ref.decode(*dev, lens, -1, SCALE, ref.FP16) if new is None else ref.runs(*dev, ctx, [n, n], -1, SCALE, weights=_weights_of([n]))
    _check(out, None, want)


@gpu
@pytest.mark.parametrize("new", [None, 2, 4, 40])
def test_small_elements_of_a_query_count_where_its_large_ones_meet_zeros(ops, new):
    """Scores made by elements 2^-27 of the query's largest, whose keys hold zero in the largest one's place."""
    H, kvh, n = 14, 2, new or 1
    ctx, lens = [50, 7], [50 + n, 7 + n]
    codes, scales, table = _pool(lens, -1, kvh, 128, 16, seed=214, spread=0.0, n_new=[n, n])
    codes.view(torch.uint8)[0, :, :, :, 0] = 0
    scales[0] = 127 + 19
    g = torch.Generator().manual_seed(215)
    q = torch.randn(2 * n, H, 128, generator=g) * 2.0 ** -27
    q[..., 0] = 1.0
    q = q.bfloat16()
    out = _attend(ops, q, codes, scales, table, lens if new is None else ctx, None if new is None else [n, n], -1)
    dev = [t.to(DEV) for t in (q, codes, scales, table)]
    want = ref.decode(*dev, lens, -1, SCALE, ref.FP16) if new is None else ref.runs(*dev, ctx, [n, n], -1, SCALE, weights=_weights_of([n]))
    _check(out, None, want)


# ------------------------------------------------------------------------------------- NaN reaches those who see it, and nobody else
def _check_with_nan(out, want):
    o, l, err_o, err_l = want
    odd = torch.isnan(o)
    assert odd.any() and torch.equal(torch.isnan(out), odd), (int((torch.isnan(out) & ~odd).sum()), int((~torch.isnan(out) & odd).sum()))
    _check(out.masked_fill(odd, 0.0), None, (o.masked_fill(odd, 0.0), l, err_o.masked_fill(odd, 0.0), err_l))


def _with_nan_values(ctx, new, wl, H, kvh, seed):
    """A cache and queries; sequence 1 has NaN codes in V at its newest token, in the middle of its run, and at the first two
    tokens of the first query's window, each in a dim and a head of its own."""
    lens = [a + b for a, b in zip(ctx, new)]
    codes, scales, table = _pool(lens, wl, kvh, 128, 16, seed=seed, spread=0.5, n_new=new)
    first = max(0, ctx[1] - wl) if wl >= 0 else 0
    for i, t in enumerate((lens[1] - 1, ctx[1] + new[1] // 2, first, first + 1)):
        row, _ = _row(codes, scales, table, 1, 1, t, i % kvh)
        row[(5, 64, 127, 0)[i]] = 0x7F if i % 2 else 0xFF
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(seed + 1)).bfloat16()
    return q, codes, scales, table


@gpu
@pytest.mark.parametrize("n,ctx,wl,H,kvh", [
    (2, 200, 64, 28, 4), (3, 200, 64, 28, 4), (4, 200, 64, 28, 4), (16, 200, 64, 28, 4), (16, 0, 5, 7, 1), (2, 31, 16, 14, 2), (5, 77, 3, 14, 2),
    (4, 200, -1, 4, 4), (13, 0, 0, 7, 1)])
def test_a_nan_value_reaches_the_queries_that_see_it_in_short_runs(ops, n, ctx, wl, H, kvh):
    ctx, new = [40, ctx, 60], [n, n, n]
    q, codes, scales, table = _with_nan_values(ctx, new, wl, H, kvh, 220)
    out = _attend(ops, q, codes, scales, table, ctx, new, wl)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, wl, SCALE, weights=ref.FP16)
    _check_with_nan(out, want)


@gpu
@pytest.mark.parametrize("n,ctx,wl,H,kvh", [
    (40, 200, 64, 28, 4), (300, 200, 64, 28, 4), (300, 200, 64, 4, 4), (20, 0, 5, 7, 1), (130, 31, -1, 14, 2), (257, 1000, 127, 8, 1), (17, 4000, 0, 6, 2)])
def test_a_nan_value_reaches_the_queries_that_see_it_in_long_runs(ops, n, ctx, wl, H, kvh):
    ctx, new = [40, ctx, 60], [n, n, n]
    q, codes, scales, table = _with_nan_values(ctx, new, wl, H, kvh, 222)
    out = _attend(ops, q, codes, scales, table, ctx, new, wl)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, wl, SCALE, weights=ref.TWO_BF16)
    _check_with_nan(out, want)


@gpu
@pytest.mark.parametrize("n", [20, 150])
def test_a_nan_key_reaches_the_queries_that_see_it_in_long_runs(ops, n):
    ctx, new, wl = [40, 90], [n, n], 64
    codes, scales, table = _pool([a + n for a in ctx], wl, 4, 128, 16, seed=224, n_new=new)
    for t in (ctx[1] + n // 2, ctx[1] - wl):
        _row(codes, scales, table, 0, 1, t, 2)[0][9] = 0x7F
    q = torch.randn(2 * n, 28, 128, generator=torch.Generator().manual_seed(225)).bfloat16()
    out = _attend(ops, q, codes, scales, table, ctx, new, wl)
    rows = torch.zeros(2 * n, 28, dtype=torch.bool)
    for i in range(n):
        pos = ctx[1] + i
        rows[n + i, 14:21] = any(pos - wl <= t <= pos for t in (ctx[1] + n // 2, ctx[1] - wl))
    assert torch.equal(torch.isnan(out).all(-1).cpu(), rows) and torch.isfinite(out.float()[~rows.to(DEV)]).all()


# ------------------------------------------------------------------------------------- lengths that go past the block table
@gpu
@pytest.mark.parametrize("new", [None, 1, 2, 5, 16, 20, 300])
@pytest.mark.parametrize("ctx,wl,H,kvh", [(500, -1, 28, 4), (390, -1, 7, 1), (500, 150, 14, 2), (395, 40, 28, 4), (900, 100, 28, 4),
                                          (3000, 2000, 4, 4), (399, 0, 7, 1)])
def test_tokens_without_a_table_entry_take_no_part(ops, new, ctx, wl, H, kvh):
    """Sequences 0 and 2 are longer than their row of the table (400 tokens; a few cases end just inside): reported, and the tokens behind it are as if they were
    not there; nothing of their neighbours gets into them."""
    n = new or 1
    ctxs, news = [ctx, 60, ctx + 7, 20], [n, min(n, 300), max(1, n - 1), n]
    lens = [a + b for a, b in zip(ctxs, news)]
    codes, scales, table = _pool(lens, wl, kvh, 128, 16, seed=230, spread=0.5, n_new=news)
    table = table[:, :25].contiguous()
    q = torch.randn(sum(news), H, 128, generator=torch.Generator().manual_seed(231)).bfloat16()
    dev = [t.to(DEV) for t in (q, codes, scales, table)]
    status = 2 if max(lens) > 400 else 0
    if new is None:
        lse = torch.empty(4, H, device=DEV)
        out = _attend(ops, q, codes, scales, table, lens, None, wl, status=status, lse=lse)
        _check(out, lse, ref.decode(*dev, lens, wl, SCALE, ref.FP16))
    else:
        out = _attend(ops, q, codes, scales, table, ctxs, news, wl, status=status)
        _check(out, None, ref.runs(*dev, ctxs, news, wl, SCALE, weights=_weights_of(news)))


@gpu
@pytest.mark.parametrize("new", [None, 1, 2, 4, 16, 40, 300])
@pytest.mark.parametrize("H,kvh,bs,wl", [(28, 4, 16, -1), (28, 4, 16, 90), (7, 1, 16, -1), (14, 2, 48, 200), (4, 4, 32, 64), (8, 1, 16, 120)])
def test_tokens_of_an_entry_outside_the_pool_take_no_part(ops, new, H, kvh, bs, wl):
    """Sequence 1 has such entries in and around its window, sequence 2 nothing else: reported, and exactly their tokens are as if
    they were not there, whichever kernel serves the run."""
    n = new or 1
    ctx, news = [300, 333, 200, 64], [n, n, n, max(1, n - 3)]
    lens = [a + b for a, b in zip(ctx, news)]
    codes, scales, table = _pool(lens, wl, kvh, 128, bs, seed=240, spread=0.5, n_new=news)
    lo = max(0, ctx[1] - wl) // bs if wl >= 0 else 0
    table[1, lo], table[1, lo + 2], table[1, (lens[1] - 1) // bs] = -1, 10 ** 6, codes.shape[1]
    table[2] = -2 ** 31
    q = torch.randn(sum(news), H, 128, generator=torch.Generator().manual_seed(241)).bfloat16()
    dev = [t.to(DEV) for t in (q, codes, scales, table)]
    if new is None:
        lse = torch.empty(4, H, device=DEV)
        out = _attend(ops, q, codes, scales, table, lens, None, wl, status=2, lse=lse)
        _check(out, lse, ref.decode(*dev, lens, wl, SCALE, ref.FP16))
    else:
        out = _attend(ops, q, codes, scales, table, ctx, news, wl, status=2)
        _check(out, None, ref.runs(*dev, ctx, news, wl, SCALE, weights=_weights_of(news)))


# ------------------------------------------------------------------------------------- block tables much wider than the sequences
def test_the_bound_on_the_lengths_bounds_the_workspace(ops):
    size = lambda mq, mb, wl, kvh=4, **kw: ops.swa_prefill_q8_workspace(3, mq, mb, kvh, 128, "meta", block_size=16, window_left=wl, **kw).numel()
    wide, tight = 65536, 20                                                # columns: 2^20 tokens, 320 tokens
    assert size(17, wide, -1) >= 2 ** 31                                   # one sequence's worth of dense rows
    assert size(17, wide, -1, max_seq_len=320) == size(17, tight, -1) < 2 ** 22
    assert size(17, wide, -1, max_seq_len=305) == size(17, tight, -1)
    assert size(17, wide, 200, max_seq_len=320) == size(17, wide, 200)     # (the window bounds them already)
    assert size(17, tight, -1, max_seq_len=10 ** 6) == size(17, tight, -1)
    assert size(4, wide, -1, max_seq_len=320) == size(4, wide, -1)         # short runs need none
    assert size(4, wide, -1, kvh=3, max_seq_len=320) == size(4, tight, -1, kvh=3)


@gpu
@pytest.mark.parametrize("wl", [-1, 50])
def test_short_sequences_behind_a_wide_table(ops, wl):
    """Sequences that do not fit the scratch together are served in turn (two at a time here), or, with a bound on their lengths, at
    once: the same values."""
    H, kvh = 28, 4
    ctx, new = [100, 0, 37, 300, 250], [20, 40, 17, 33, 18]
    lens = [a + b for a, b in zip(ctx, new)]
    codes, scales, table = _pool(lens, -1, kvh, 128, 16, seed=250, spread=0.5, n_new=new)
    table = torch.cat([table, torch.full((5, 4096 - table.shape[1]), -1, dtype=torch.int32)], 1)
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(251)).bfloat16()
    plain = _attend(ops, q, codes, scales, table, ctx, new, wl)
    bound = _attend(ops, q, codes, scales, table, ctx, new, wl, max_seq_len=max(lens))
    ws = ops.swa_prefill_q8_workspace(5, 40, 4096, kvh, 128, DEV, block_size=16, window_left=wl, max_seq_len=max(lens))
    given = _attend(ops, q, codes, scales, table, ctx, new, wl, max_seq_len=max(lens), workspace=ws)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, wl, SCALE, weights=ref.TWO_BF16)
    _check(plain, None, want)
    assert torch.equal(bound, plain) and torch.equal(given, plain)
    # a bound that does not hold: reported
    if wl < 0:
        short = _attend(ops, q, codes, scales, table, ctx, new, wl, max_seq_len=320, status=2)
        keep = torch.ones(sum(new), dtype=torch.bool, device=DEV)
        keep[77 + 20:77 + 33] = False                                      # the queries of sequence 3 behind token 320
        assert torch.equal(short[keep], plain[keep])


@gpu
def test_backend_prompt_behind_a_wide_table_takes_little_memory(ops):
    from tests.test_kv_q8 import _impl, _meta
    H, kvh, D, bs = 28, 4, 128, 16
    ctx, new = [30, 0], [50, 20]
    impl = _impl(window=None)
    table = torch.full((2, 8192), -1, dtype=torch.int32, device=DEV)       # room for 131072 tokens each
    table[0, :6], table[1, :6] = torch.arange(6, device=DEV), torch.arange(6, 12, device=DEV)
    kv, sc = ops.kv_cache_q8(12, bs, kvh, D, device=DEV)
    slots = torch.cat([torch.arange(30, 80, device=DEV), 96 + torch.arange(20, device=DEV)])
    old = torch.cat([torch.arange(30, device=DEV)])
    k0, v0 = (_rows((30, kvh, D), 260 + i).bfloat16().to(DEV) for i in range(2))
    ops.kv_append_q8(k0, v0, kv[0], kv[1], sc[0], sc[1], old)
    q, k, v = (_rows((70, h, D), 262 + i).bfloat16().to(DEV) for i, h in enumerate((H, kvh, kvh)))
    out = torch.empty(70, H * D, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    impl.forward(None, q, k, v, None, None, None, kv, _meta(ctx, new, 2, table, slots, DEV), output=out, kv_scales=sc)
    assert torch.cuda.max_memory_allocated() - before < 8 * 2 ** 20
    assert impl.status() == 0
    _check(out.view(70, H, D), None, ref.runs(q, kv, sc, table, ctx, new, -1, D ** -0.5, weights=ref.TWO_BF16))


A = 1 << 20          # an aligned address that is never dereferenced: the calls below are refused on the host


@pytest.mark.parametrize("blocks,block", [(2 ** 26 + 1, 16), (32768, 65536), (2 ** 31 - 1, 16), (2 ** 30 // 48 + 1, 48)])
def test_tables_beyond_32_bit_positions_are_refused(sb, blocks, block):
    from spikingbrain_7b_b200 import _abi
    scale, cs, ss = ctypes.c_float(0.1), 4 * 128 * block, 4 * block
    assert _abi.lib.sbk_swa_decode_q8(A, 3584, A, A, A, A, A, blocks, A, 2, 28, 4, 128, 8, block, cs, ss, 15, scale, A, 0, 3584, None, A,
                                      1 << 40, None, None) == -1
    assert b"2^30" in _abi.lib.sbk_last_error()
    for most in (5, 40):
        assert _abi.lib.sbk_swa_prefill_q8(A, 3584, A, A, A, A, A, blocks, A, A, 2, most, 28, 4, 128, 8, block, cs, ss, 15, scale, A, 3584, A,
                                           1 << 40, None, None) == -1
        assert b"2^30" in _abi.lib.sbk_last_error()


@gpu
@pytest.mark.parametrize("new", [None, 3, 20])
def test_the_last_positions_of_the_widest_table(ops, new):
    """2^30 tokens of room; one sequence that fills it, one that claims 2^31 - 1 (clamped to 2^30 tokens of context in runs)."""
    H, kvh, bs, n, wl = 7, 1, 65536, new or 1, 40
    g = torch.Generator().manual_seed(270)
    codes = torch.randn(2, 2, bs, kvh, 128, generator=g).to(torch.float8_e4m3fn)
    scales = torch.full((2, 2, kvh, bs), 126, dtype=torch.uint8)
    table = torch.full((2, 16384), -1, dtype=torch.int32)
    table[:, -1] = 1
    ctx = [2 ** 30 - n, 2 ** 31 - 1 - n]
    q = torch.randn(2 * n, H, 128, generator=g).bfloat16()
    dev = [t.to(DEV) for t in (q, codes, scales, table)]
    if new is None:
        out = _attend(ops, q, codes, scales, table, [2 ** 30, 2 ** 31 - 1], None, wl, status=2)
        want = ref.decode(*dev, [2 ** 30, 2 ** 31 - 1], wl, SCALE, ref.FP16)
    else:
        out = _attend(ops, q, codes, scales, table, ctx, [n, n], wl, status=2)
        want = ref.runs(*dev, [ctx[0], 2 ** 30], [n, n], wl, SCALE, weights=_weights_of([n]))
    _check(out, None, want)


def test_overlapping_output_rows_are_refused(sb):
    from spikingbrain_7b_b200 import _abi
    decode = lambda B, stride: _abi.lib.sbk_swa_decode_q8(A, 3584, A, A, A, A, A, 4, A, B, 28, 4, 128, 8, 16, 8192, 64, 15, ctypes.c_float(0.1), A, 0,
                                                          stride, None, None, 0, None, None)
    assert decode(2, 0) == decode(2, 3576) == -1 and b"overlap" in _abi.lib.sbk_last_error()
    assert decode(1, 0) == decode(2, 3584) == -3                           # (the next check: no workspace)
    for most in (5, 40):
        assert _abi.lib.sbk_swa_prefill_q8(A, 3584, A, A, A, A, A, 4, A, A, 2, most, 28, 4, 128, 8, 16, 8192, 64, 15, ctypes.c_float(0.1), A, 0,
                                           None, 0, None, None) == -1
        assert b"overlap" in _abi.lib.sbk_last_error()


@gpu
def test_calls_without_queries_give_empty_outputs(ops):
    kv, sc = ops.kv_cache_q8(4, 16, 4, 128, device=DEV)
    table = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 28, 128, dtype=torch.bfloat16, device=DEV)
    for most in (0, 1, 40):
        out = ops.swa_prefill_q8(q, kv[0], kv[1], sc[0], sc[1], table, _i32(0, 0, 0), _i32(3, 5), most, window_left=-1)
        assert out.shape == (0, 28, 128)
    assert ops.swa_decode_q8(q, kv[0], kv[1], sc[0], sc[1], table[:0], _i32(), window_left=-1).shape == (0, 28, 128)


@gpu
@pytest.mark.parametrize("new", [None, 4, 40])
def test_repeated_calls_on_two_streams_and_from_two_graphs_give_the_same_bits(ops, new):
    """No atomics whose order changes a sum, no workspace shared between calls that may overlap."""
    H, kvh, n = 28, 4, new or 1
    ctx = [3000, 200, 5000, 0, 1111]
    lens = [c + n for c in ctx]
    codes, scales, table = (t.to(DEV) for t in _pool(lens, 2000, kvh, 128, 16, seed=280, n_new=[n] * 5))
    qs = [_rows((5 * n, H, 128), 281 + i).bfloat16().to(DEV) for i in range(2)]
    lens_d, ctx_d, start = _i32(*lens), _i32(*ctx), _starts([n] * 5)

    def call(i):
        if new is None:
            return ops.swa_decode_q8(qs[i], *codes, *scales, table, lens_d, window_left=2000)
        return ops.swa_prefill_q8(qs[i], *codes, *scales, table, start, ctx_d, n, window_left=2000)
    want = [call(i).clone() for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(call(i))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        eager = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
                eager.append(call(i))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i]) and torch.equal(eager[i], want[i])
            outs[i].fill_(0.0)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["auto", "fp8_e4m3"])
def test_backend_says_why_it_takes_no_calibrated_scales(sb, dtype):
    from types import SimpleNamespace
    from tests.test_kv_q8 import _impl, _meta
    q, k = torch.zeros(1, 28, 128).bfloat16(), torch.zeros(1, 4, 128).bfloat16()
    md = _meta([3], [1], 0, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), "cpu")
    with pytest.raises(AssertionError, match="one scale per tensor"):
        _impl(dtype).forward(SimpleNamespace(_k_scale_float=0.5, _v_scale_float=1.0), q, k, k, None, None, None,
                             torch.zeros(2, 4, 16, 4, 128, dtype=torch.uint8), md, output=torch.empty_like(q))


@gpu
@pytest.mark.parametrize("lens,wl,H,kvh", [([1, 17, 300, 2050, 0], 1024, 28, 4), ([30011, 6000], -1, 7, 1), ([8193] * 3, 4096, 14, 2),
                                           ([1500] * 160, 1000, 28, 4)])
def test_single_tokens_hold_their_weights_in_fp16(ops, lens, wl, H, kvh):
    codes, scales, table = _pool(lens, wl, kvh, 128, 16, seed=290, spread=0.5)
    q = torch.randn(len(lens), H, 128, generator=torch.Generator().manual_seed(291)).bfloat16()
    want = ref.decode(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), lens, wl, SCALE, ref.FP16)
    for dtype in (torch.float32, torch.bfloat16):
        lse = torch.empty(len(lens), H, device=DEV)
        out = _attend(ops, q, codes, scales, table, lens, None, wl, out_dtype=dtype, lse=lse)
        _check(out, lse, want)
        assert mean_rel(out.float(), want[0].to(dtype).float()) <= MEAN_REL


@gpu
@pytest.mark.parametrize("ctx,new,wl,H,kvh", [([4200] * 8, [4] * 8, 4096, 28, 4), ([30000, 7], [16, 5], -1, 7, 1), ([900, 0, 2000], [2, 1, 2], 700, 14, 2)])
def test_short_runs_hold_their_weights_in_fp16(ops, ctx, new, wl, H, kvh):
    lens = [a + b for a, b in zip(ctx, new)]
    codes, scales, table = _pool(lens, wl, kvh, 128, 16, seed=292, spread=0.5, n_new=new)
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(293)).bfloat16()
    out = _attend(ops, q, codes, scales, table, ctx, new, wl)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, wl, SCALE, weights=ref.FP16)
    _check(out, None, want)
    assert mean_rel(out.float(), want[0].bfloat16().float()) <= MEAN_REL


@gpu
@pytest.mark.parametrize("H,kvh", [(6, 3), (5, 5), (64, 8), (12, 6)])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 0, 9], [40, 3, 300]])
def test_runs_with_other_numbers_of_kv_heads(ops, H, kvh, new):
    ctx = [100, 7, 0]
    codes, scales, table = _pool([a + b for a, b in zip(ctx, new)], 90, kvh, 128, 32, seed=300, spread=0.5, n_new=new)
    q = torch.randn(sum(new), H, 128, generator=torch.Generator().manual_seed(301)).bfloat16()
    out = _attend(ops, q, codes, scales, table, ctx, new, 90)
    want = ref.runs(q.to(DEV), codes.to(DEV), scales.to(DEV), table.to(DEV), ctx, new, 90, SCALE, weights=ref.TWO_BF16)
    _check(out, None, want)


@gpu
@pytest.mark.parametrize("new", [None, 4, 40])
def test_infinite_queries_spoil_their_own_rows_only(ops, new):
    """Scores of +-inf and NaN stay in the rows whose query makes them, the other heads and queries of their tiles keep their values."""
    H, kvh, n = 14, 2, new or 1
    ctx, lens = [60, 300], [60 + n, 300 + n]
    codes, scales, table = _pool(lens, 100, kvh, 128, 16, seed=302, spread=0.5, n_new=[n, n])
    q = torch.randn(2 * n, H, 128, generator=torch.Generator().manual_seed(303)).bfloat16()
    clean = q.clone()
    q[0, 3, 5], q[n, 9, 127], q[2 * n - 1, 0, 0] = math.inf, -math.inf, math.nan
    spoilt = torch.zeros(2 * n, H, dtype=torch.bool, device=DEV)
    spoilt[0, 3] = spoilt[n, 9] = spoilt[2 * n - 1, 0] = True
    args = (codes, scales, table, lens if new is None else ctx, None if new is None else [n, n], 100)
    a, b = _attend(ops, q, *args), _attend(ops, clean, *args)
    assert torch.equal(a[~spoilt], b[~spoilt]) and not torch.isfinite(a.float()[spoilt]).all(-1).any()
