"""The 8-bit paged K/V cache: quantising append, read-back and attention against their definitions in 64 bits
(oracle/kv_q8.py)."""
import ctypes
import math

import pytest
import torch

from oracle import kv_q8 as ref
from oracle import ref_ops

DEV = "cuda:0"
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(sb):
    from spikingbrain_7b_b200 import ops as o
    return o


def _status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _rows(shape, seed, spread=3.0):
    """Normal rows, each with a magnitude of its own (over a factor of about e^spread)."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * torch.exp(spread * (torch.rand(shape[:-1] + (1,), generator=g) - 0.5))


def _odd_rows(D):
    """Rows at the edges of the format."""
    r = [torch.zeros(D), torch.full((D,), 448.0), torch.full((D,), 448.0 * (1 + 2.0 ** -7)), torch.full((D,), 2.0 ** -90),
         torch.full((D,), 3.0e38), torch.full((D,), -448.0 * 2.0 ** 63), torch.full((D,), 1e-44)]
    x = torch.linspace(-1.0, 1.0, D)
    r += [x, x * 448.0, x * 449.0, x * 2.0 ** 60, x * 2.0 ** 70, x * 2.0 ** -60, x * 2.0 ** -70]
    for bad in (math.inf, -math.inf, math.nan):
        y = x.clone()
        y[3], y[D - 1] = bad, bad
        r.append(y)
    r.append(torch.full((D,), math.nan))
    ties = torch.tensor([1.0 + i / 16 for i in range(16)] + [448.0])        # half-way points between codes
    y = torch.zeros(D)
    y[:17] = ties
    r.append(y)
    return torch.stack(r)


# ------------------------------------------------------------------------------------- CPU: the oracle and the refusals
def test_oracle_codes_are_torch_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    v = ref.code_values()
    assert torch.equal(torch.isnan(t), torch.isnan(v)) and torch.equal(t.nan_to_num(0), v.nan_to_num(0))
    x = torch.linspace(-448, 448, 40001).double()[:, None]                   # fp32 numbers: both sides see the same ones
    x = torch.cat([x, torch.full_like(x, 448.0)], 1)                        # pins the exponent at 0
    c, b = ref.quantise(x)
    assert (b == 127).all()
    assert torch.equal(c[:, 0].view(torch.float8_e4m3fn).float(), x[:, 0].float().to(torch.float8_e4m3fn).float())


def test_oracle_row_exponent_is_the_smallest_that_fits():
    x = _odd_rows(64)
    c, b = ref.quantise(x)
    e = b.long() - 127
    for row, k in zip(x.double(), e.tolist()):
        top = float(row[torch.isfinite(row)].abs().max()) if torch.isfinite(row).any() else 0.0
        assert top <= 448 * 2.0 ** k or k == 63
        assert k == -64 or top > 448 * 2.0 ** (k - 1)
    v = ref.values(c, b)
    fine = torch.isfinite(x)
    assert torch.equal(torch.isnan(v), ~fine)
    assert torch.equal(v[fine].float().bfloat16().double(), v[fine])        # every value is a bf16 number


def test_entry_points_take_cuda_tensors_only(ops):
    kv, sc = ops.kv_cache_q8(4, 16, 2, 128, device="cpu")
    assert kv.shape == (2, 4, 16, 2, 128) and kv.dtype == torch.float8_e4m3fn
    assert sc.shape == (2, 4, 2, 16) and sc.dtype == torch.uint8 and (sc == 63).all()
    with pytest.raises(ValueError):
        ops.kv_cache_q8(4, 24, 2, 128, device="cpu")
    k = torch.zeros(3, 2, 128)
    slots = torch.zeros(3, dtype=torch.int64)
    tab, lens = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.kv_append_q8(k, k, kv[0], kv[1], sc[0], sc[1], slots)
    with pytest.raises(RuntimeError):
        ops.rope_kv_append_q8(None, k, k, kv[0], kv[1], sc[0], sc[1], slots, slots, torch.zeros(8, 128))
    with pytest.raises(RuntimeError):
        ops.kv_gather_q8(kv[0], kv[1], sc[0], sc[1], tab, lens, 4)
    with pytest.raises(RuntimeError):
        ops.swa_decode_q8(torch.zeros(1, 4, 128).bfloat16(), kv[0], kv[1], sc[0], sc[1], tab, lens, window_left=4)
    with pytest.raises(RuntimeError):
        ops.swa_prefill_q8(torch.zeros(1, 4, 128).bfloat16(), kv[0], kv[1], sc[0], sc[1], tab,
                           torch.zeros(2, dtype=torch.int32), lens, 1, window_left=4)


A = 1 << 20          # an aligned address that is never dereferenced: every call below is refused on the host


def _append_args(**over):
    a = dict(key=A, value=A, dtype=0, k_cache=A, v_cache=A, k_scale=A, v_scale=A, slots=A, T=2, kvh=4, D=128,
             tok=1024, nb=8, bs=16, cs=8192, ss=64, tables=None, max_blocks=0, lens=None, qsl=None, B=0, wl=-1, ret=None,
             max_ret=0, status=None, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(T=-1), -1), (dict(dtype=2), -1), (dict(D=96), -1), (dict(kvh=0), -1), (dict(bs=24), -1), (dict(bs=0), -1),
    (dict(k_scale=None), -1), (dict(k_cache=None), -1), (dict(key=None), -1), (dict(slots=None), -1),
    (dict(key=A + 8), -2), (dict(k_cache=A + 8), -2), (dict(v_scale=A + 4), -2), (dict(tok=1032), -2), (dict(cs=8200), -2),
    (dict(ss=72), -2), (dict(tok=512), -1), (dict(cs=4096), -1), (dict(ss=48), -1),
    (dict(tables=A, B=2, lens=None, max_blocks=4), -1), (dict(tables=A, B=2, lens=A, max_blocks=0), -1),
    (dict(tables=A, B=2, lens=A, max_blocks=4, ret=A, max_ret=0), -1)])
def test_append_refusals(sb, over, code):
    from spikingbrain_7b_b200 import _abi
    assert _abi.lib.sbk_kv_append_q8(*_append_args(**over)) == code
    assert b"sbk_kv_append_q8" in _abi.lib.sbk_last_error()


@pytest.mark.parametrize("over,code", [
    (dict(rot=24), -1), (dict(rot=0), -1), (dict(rot=144), -1), (dict(pos=None), -1), (dict(tab=None), -1),
    (dict(max_pos=0), -1), (dict(tab=A + 8), -2), (dict(q=A + 8), -2), (dict(qs=7176), -2), (dict(qs=1024), -1),
    (dict(H=0), -1), (dict(H=-1), -1), (dict(D=80), -1)])
def test_rope_append_refusals(sb, over, code):
    from spikingbrain_7b_b200 import _abi
    a = dict(q=A, H=28, qs=7168, key=A, value=A, in_place=0, dtype=0, k_cache=A, v_cache=A, k_scale=A, v_scale=A, slots=A,
             pos=A, tab=A, rot=128, max_pos=64, T=2, kvh=4, D=128, tok=1024, nb=8, bs=16, cs=8192, ss=64, tables=None,
             max_blocks=0, lens=None, qsl=None, B=0, wl=-1, ret=None, max_ret=0, status=None, stream=None)
    a.update(over)
    assert _abi.lib.sbk_rope_kv_append_q8(*a.values()) == code
    assert b"sbk_rope_kv_append_q8" in _abi.lib.sbk_last_error()


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), -1), (dict(B=65536), -1), (dict(n_out=-1), -1), (dict(dt=7), -1), (dict(D=32), -1), (dict(bs=20), -1),
    (dict(lens=None), -1), (dict(ko=None), -1), (dict(ko=A + 8), -2), (dict(ss=65), -2), (dict(max_blocks=0), -1)])
def test_gather_refusals(sb, over, code):
    from spikingbrain_7b_b200 import _abi
    a = dict(k=A, v=A, ks=A, vs=A, tables=A, max_blocks=4, lens=A, B=2, kvh=4, D=128, nb=8, bs=16, cs=8192, ss=64, wl=-1,
             ko=A, vo=A, dt=0, n_out=5, status=None, stream=None)
    a.update(over)
    assert _abi.lib.sbk_kv_gather_q8(*a.values()) == code


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), -1), (dict(H=30), -1), (dict(H=36), -1), (dict(kvh=3, H=27), -1), (dict(D=64), -1), (dict(bs=8), -1),
    (dict(max_blocks=0), -1), (dict(dt=5), -1), (dict(q=None), -1), (dict(lens=None), -1), (dict(vs=None), -1),
    (dict(q=A + 2), -2), (dict(qs=3585), -2), (dict(k=A + 8), -2), (dict(ks=A + 8), -2), (dict(cs=8200), -2),
    (dict(cs=4096), -1), (dict(ss=16), -1)])
def test_decode_refusals(sb, over, code):
    from spikingbrain_7b_b200 import _abi
    a = dict(q=A, qs=3584, k=A, v=A, ks=A, vs=A, tables=A, max_blocks=4, lens=A, B=2, H=28, kvh=4, D=128, nb=8, bs=16,
             cs=8192, ss=64, wl=-1, scale=ctypes.c_float(0.1), out=A, dt=0, os=3584, lse=None, ws=A, wsb=1 << 40,
             status=None, stream=None)
    a.update(over)
    assert _abi.lib.sbk_swa_decode_q8(*a.values()) == code
    assert b"sbk_swa_decode_q8" in _abi.lib.sbk_last_error()


@pytest.mark.parametrize("over,code", [
    (dict(n=-1), -1), (dict(mq=-1), -1), (dict(H=30), -1), (dict(H=36), -1), (dict(D=64), -1), (dict(bs=8), -1),
    (dict(q=None), -1), (dict(qsl=None), -1), (dict(ctx=None), -1), (dict(k=A + 8), -2), (dict(cs=4096), -1)])
def test_prefill_refusals(sb, over, code):
    from spikingbrain_7b_b200 import _abi
    a = dict(q=A, qs=3584, k=A, v=A, ks=A, vs=A, tables=A, max_blocks=4, qsl=A, ctx=A, n=2, mq=5, H=28, kvh=4, D=128, nb=8,
             bs=16, cs=8192, ss=64, wl=-1, scale=ctypes.c_float(0.1), out=A, os=3584, ws=A, wsb=1 << 40, status=None,
             stream=None)
    a.update(over)
    assert _abi.lib.sbk_swa_prefill_q8(*a.values()) == code
    assert b"sbk_swa_prefill_q8" in _abi.lib.sbk_last_error()


def test_calls_without_work_succeed(sb):
    from spikingbrain_7b_b200 import _abi
    assert _abi.lib.sbk_kv_append_q8(*_append_args(T=0, key=None, value=None, slots=None)) == 0


# ------------------------------------------------------------------------------------- append and read-back
@gpu
@pytest.mark.parametrize("dtype,kvh,D,bs", [(torch.bfloat16, 4, 128, 16), (torch.float32, 2, 64, 32),
                                            (torch.bfloat16, 3, 256, 16), (torch.float32, 1, 128, 48),
                                            (torch.bfloat16, 1, 64, 16)])
def test_append_stores_the_definition_bit_for_bit(ops, dtype, kvh, D, bs):
    odd = _odd_rows(D)
    T, nb = 61, 9
    k, v = _rows((T, kvh, D), 1), _rows((T, kvh, D), 2, 30.0)
    k[:odd.shape[0], kvh - 1] = odd
    v[T - odd.shape[0]:, 0] = odd
    k, v = k.to(dtype), v.to(dtype)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(nb * bs, generator=g)[:T]
    slots[5] = slots[40] = -1
    kv, sc = ops.kv_cache_q8(nb, bs, kvh, D, device=DEV)
    kv.view(torch.uint8).fill_(0x5A)
    sc.fill_(9)
    st = _status()
    ops.kv_append_q8(k.to(DEV), v.to(DEV), kv[0], kv[1], sc[0], sc[1], slots.to(DEV), status=st)
    assert st.item() == 0
    want_c = torch.full((2, nb * bs, kvh, D), 0x5A, dtype=torch.uint8)
    want_s = torch.full((2, nb, kvh, bs), 9, dtype=torch.uint8)
    for j, x in enumerate((k, v)):
        c, b = ref.quantise(x)
        for t, slot in enumerate(slots.tolist()):
            if slot >= 0:
                want_c[j, slot] = c[t]
                want_s[j, slot // bs, :, slot % bs] = b[t]
    got_c = kv.view(torch.uint8).cpu().view(2, nb * bs, kvh, D)
    nan = (want_c & 127) == 127                                              # NaN codes: either sign
    assert torch.equal((got_c & 127)[nan], (want_c & 127)[nan]) and torch.equal(got_c[~nan], want_c[~nan])
    assert torch.equal(sc.cpu(), want_s)


@gpu
def test_append_strided_views_bad_slots_and_retirement(ops):
    kvh, D, bs, nb = 4, 128, 16, 12
    qkv = _rows((5, 36, D), 4).bfloat16().to(DEV)                            # a fused projection: K and V are strided views
    k, v = qkv[:, 28:32], qkv[:, 32:36]
    kv, sc = ops.kv_cache_q8(nb, bs, kvh, D, device=DEV)
    table = torch.arange(10, dtype=torch.int32, device=DEV).view(1, 10).contiguous()
    retired = torch.full((1, 4), -7, dtype=torch.int32, device=DEV)
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    qsl = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    st = _status()
    slots = torch.tensor([95, 96, 97, nb * bs, 99], device=DEV)
    ops.kv_append_q8(k, v, kv[0], kv[1], sc[0], sc[1], slots, block_tables=table, seq_lens=lens, query_start_loc=qsl,
                     window_left=40, retired_out=retired, status=st)
    assert st.item() == 1                                                    # SBK_ST_BAD_SLOT, the others are written
    for t, slot in ((0, 95), (1, 96), (2, 97), (4, 99)):
        c, b = ref.quantise(k[t])
        assert torch.equal(kv[0].view(torch.uint8)[slot // bs, slot % bs].cpu(), c)
        assert torch.equal(sc[0][slot // bs, :, slot % bs].cpu(), b)
    assert table.cpu().tolist()[0][:4] == [-1, -1, -1, 3] and retired.cpu().tolist()[0] == [0, 1, 2, -1]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot_dim,H,kvh", [(128, 128, 28, 4), (128, 64, 7, 1), (64, 32, 4, 2), (256, 256, 2, 1), (128, 16, 3, 3)])
def test_rope_append_against_64_bits(ops, dtype, D, rot_dim, H, kvh):
    T, bs, nb, max_pos = 45, 16, 7, 5000
    q, k, v = (_rows((T, n, D), 10 + i).to(dtype) for i, n in enumerate((H, kvh, kvh)))
    table = ops.build_cos_sin_cache(rot_dim, max_pos, 10000.0, dtype, device="cpu")
    g = torch.Generator().manual_seed(5)
    pos = torch.randint(0, max_pos, (T,), generator=g)
    slots = torch.randperm(nb * bs, generator=g)[:T]
    slots[3] = -1                                                            # still rotated, not written
    pos[7] = max_pos                                                         # untouched
    qd, kd = q.to(DEV), k.to(DEV)
    kv, sc = ops.kv_cache_q8(nb, bs, kvh, D, device=DEV)
    st = _status()
    ops.rope_kv_append_q8(qd, kd, v.to(DEV), kv[0], kv[1], sc[0], sc[1], slots.to(DEV), pos.to(DEV), table.to(DEV),
                          key_in_place=True, status=st)
    assert st.item() == 16                                                   # SBK_ST_BAD_POSITION
    half = rot_dim // 2
    pc = pos.clamp(max=max_pos - 1)
    c, s = table.double()[pc][:, None, :half], table.double()[pc][:, None, half:]

    def turn(x):
        x = x.double()
        a, b, rest = x[..., :half], x[..., half:rot_dim], x[..., rot_dim:]
        mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), torch.zeros_like(rest)], -1)
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1), mag * 2.0 ** -23   # two products and a sum in fp32
    live = torch.ones(T, dtype=torch.bool)
    live[7] = False
    step = torch.finfo(dtype).eps / 2
    for got, x in ((qd, q), (kd, k)):
        want, err = turn(x)
        bound = err * (1 + step) + step * want.abs() + 1e-40
        assert ((got.cpu().double() - want).abs() <= bound)[live].all()
        assert torch.equal(got.cpu()[7], x[7])
    want, err = turn(k)
    flat = kv.view(2, nb * bs, kvh, D)
    for t in range(T):
        if t in (3, 7):
            continue
        slot = int(slots[t])
        byte = sc[:, slot // bs, :, slot % bs].cpu()
        got = ref.values(flat[:, slot].cpu(), byte)
        # nearest code of a value that is off by err: half a step of the value, or of the smallest codes (2^-9)
        low = 2.0 ** -10 * 2.0 ** (byte.double() - 127).unsqueeze(-1)
        bound = torch.maximum((want[t].abs() + err[t]) * 2.0 ** -4, low[0]) + err[t]
        assert ((got[0] - want[t]).abs() <= bound).all()
        e = byte[0].double() - 127
        top = want[t].abs().amax(-1)
        assert (top <= 448 * 2.0 ** e * (1 + 2.0 ** -21)).all() and (top >= 448 * 2.0 ** (e - 1) * (1 - 2.0 ** -21)).all()
        cv, bv = ref.quantise(v[t])
        assert torch.equal(flat[1, slot].view(torch.uint8).cpu(), cv) and torch.equal(byte[1], bv)
    for t in (3, 7):
        assert slots[t] == -1 or (flat[:, int(slots[t])].view(torch.uint8) == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kvh,D,bs,wl", [(4, 128, 16, 100), (2, 64, 32, -1), (1, 256, 16, 0)])
def test_gather_returns_the_values_exactly(ops, dtype, kvh, D, bs, wl):
    lens = [1, 16, 17, 0, 64, 65, 200, 333]
    codes, scales, table = _pool(lens, wl, kvh, D, bs, seed=6)
    n_out = max(1, max(min(L, wl + 1) if wl >= 0 else L for L in lens)) + 3
    st = _status()
    k, v = ops.kv_gather_q8(codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV), table.to(DEV),
                            torch.tensor(lens, dtype=torch.int32, device=DEV), n_out, window_left=wl, dtype=dtype, status=st)
    assert st.item() == 0 and k.dtype == dtype and k.shape == (len(lens), kvh, n_out, D)
    for b, L in enumerate(lens):
        t0 = ref_ops.first_visible(L, 1, wl)
        for j, got in enumerate((k, v)):
            want = ref.window_values(codes[j], scales[j], table[b], t0, L).transpose(0, 1)
            assert torch.equal(got[b, :, :L - t0].cpu().double(), want)
            assert not got[b, :, L - t0:].any()


@gpu
def test_gather_reports_a_bad_block_and_keeps_the_rest(ops):
    codes, scales, table = _pool([40, 40], -1, 2, 128, 16, seed=7)
    table[1, 1] = 10 ** 6
    st = _status()
    k, _ = ops.kv_gather_q8(codes[0].to(DEV), codes[1].to(DEV), scales[0].to(DEV), scales[1].to(DEV), table.to(DEV),
                            torch.tensor([40, 40], dtype=torch.int32, device=DEV), 40, status=st)
    assert st.item() == 2 and not k[1, :, 16:32].any() and k[1, :, 32:].any()
    assert torch.equal(k[0].cpu().double(), ref.window_values(codes[0], scales[0], table[0], 0, 40).transpose(0, 1))


# ------------------------------------------------------------------------------------- attention
def _pool(lens, wl, kvh, D, bs, seed, spread=3.0, slack=5, n_new=None):
    """A cache that holds the visible tokens behind a permuted table. Everything nobody wrote (other blocks, the tail of the
    newest one, its exponents) holds NaN codes and the largest exponent."""
    g = torch.Generator().manual_seed(seed)
    n_new = n_new or [1] * len(lens)
    first = [ref_ops.first_visible(L, n, wl) // bs for L, n in zip(lens, n_new)]
    last = [-(-L // bs) for L in lens]
    nb = sum(b - a for a, b in zip(first, last)) + slack
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(last))), -1, dtype=torch.int32)
    codes = torch.full((2, nb, bs, kvh, D), 0x7F, dtype=torch.uint8)
    scales = torch.full((2, nb, kvh, bs), 190, dtype=torch.uint8)
    o = 0
    for b, L in enumerate(lens):
        n = last[b] - first[b]
        if n <= 0:
            continue
        ids = perm[o:o + n]
        o += n
        table[b, first[b]:last[b]] = ids
        x = torch.randn(2, n, bs, kvh, D, generator=g) * torch.exp(spread * (torch.rand(2, n, bs, kvh, 1, generator=g) - 0.5))
        m, k = torch.frexp(x.abs().amax(-1))
        e = (k - 9 + (m > 0.875).int()).clamp(-64, 63)
        c = torch.ldexp(x, -e.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
        s = (e + 127).to(torch.uint8).transpose(2, 3).contiguous()
        tail = L - (last[b] - 1) * bs
        c[:, -1, tail:] = 0x7F
        s[:, -1, :, tail:] = 190
        codes[:, ids.long()], scales[:, ids.long()] = c, s
    return codes.view(torch.float8_e4m3fn), scales, table


def _check(out, lse, want):
    o, l, err_o, err_l = want
    half = torch.finfo(out.dtype).eps / 2
    bound = err_o * (1 + half) + half * o.abs() + 1e-30
    off = (out.double() - o).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= bound).all(), (float((off / bound).max()), float(off.max()))
    if lse is not None:
        fin = torch.isfinite(l)
        assert torch.equal(torch.isfinite(lse), fin) and (lse[~fin] == -math.inf).all()
        assert ((lse.double() - l).abs()[fin] <= err_l[fin]).all(), float(((lse.double() - l).abs()[fin] / err_l[fin]).max())


def _decode(ops, lens, wl, H, kvh, bs, seed, out_dtype=torch.bfloat16, spread=3.0, scale=None, qmag=1.0, workspace=None):
    codes, scales, table = _pool(lens, wl, kvh, 128, bs, seed, spread)
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    q = (qmag * _rows((len(lens), H, 128), seed + 1)).bfloat16().to(DEV)
    st = _status()
    lse = torch.empty(len(lens), H, device=DEV)
    scale = 128 ** -0.5 if scale is None else scale
    out = ops.swa_decode_q8(q, codes[0], codes[1], scales[0], scales[1], table,
                            torch.tensor(lens, dtype=torch.int32, device=DEV), window_left=wl, lse=lse, out_dtype=out_dtype,
                            scale=scale, status=st, workspace=workspace)
    assert st.item() == 0
    want = ref.decode(q, codes, scales, table, lens, wl, scale)
    _check(out, lse, want)
    return out


@gpu
@pytest.mark.parametrize("lens", [[1], [2], [16], [17], [15, 31, 33, 0], [64, 65, 66, 127, 128, 129], [0], [0, 0, 5]])
def test_decode_small_lengths(ops, lens):
    _decode(ops, lens, 4096, 28, 4, 16, seed=20)


@gpu
@pytest.mark.parametrize("wl", [0, 1, 15, 16, 17, 31, 32, 4095, 4096, -1])
def test_decode_windows(ops, wl):
    _decode(ops, [1, 33, 4500, 700, 4097], wl, 28, 4, 16, seed=21)


@gpu
@pytest.mark.parametrize("H,kvh", [(7, 1), (8, 1), (1, 1), (14, 2), (6, 2), (28, 4), (32, 4), (4, 4), (8, 4)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_decode_head_layouts(ops, H, kvh, out_dtype):
    _decode(ops, [300, 1, 1025, 77, 48], 500, H, kvh, 16, seed=22, out_dtype=out_dtype)


@gpu
@pytest.mark.parametrize("bs", [16, 32, 48, 128, 256])
def test_decode_block_sizes(ops, bs):
    _decode(ops, [300, 1, 1025, 77, 48, 2049], 600, 14, 2, bs, seed=23)


@gpu
@pytest.mark.parametrize("lens,H,kvh", [([8193], 28, 4), ([8193, 5000, 4097], 28, 4), ([30011], 7, 1), ([6000, 20001], 14, 2)])
def test_decode_few_long_sequences(ops, lens, H, kvh):
    _decode(ops, lens, 4096, H, kvh, 16, seed=24)
    _decode(ops, lens, -1, H, kvh, 16, seed=25)


@gpu
@pytest.mark.parametrize("n,H,kvh", [(300, 28, 4), (1024, 7, 1), (1025, 4, 2), (2100, 2, 1)])
def test_decode_many_sequences(ops, n, H, kvh):
    g = torch.Generator().manual_seed(26)
    lens = (torch.exp(torch.rand(n, generator=g) * math.log(700.0))).long().tolist()
    lens[0], lens[n // 2], lens[n - 1] = 0, 3000, 0
    _decode(ops, lens, 400, H, kvh, 16, seed=27)


@gpu
def test_decode_equal_sequences_that_fill_the_gpu(ops):
    _decode(ops, [1500] * 160, 1000, 28, 4, 16, seed=28)


@gpu
@pytest.mark.parametrize("spread,qmag,scale", [(60.0, 1.0, None), (0.0, 60.0, None), (3.0, 1e-3, None), (3.0, 1.0, 0.0),
                                               (3.0, 1.0, -0.3), (3.0, 300.0, 1e-3)])
def test_decode_magnitudes(ops, spread, qmag, scale):
    """Rows of very different scale, peaked and flat softmaxes, a zero and a negative scale."""
    _decode(ops, [700, 33, 2050], 1024, 28, 4, 16, seed=29, spread=spread, qmag=qmag, scale=scale, out_dtype=torch.float32)


@gpu
def test_decode_strided_rows_and_workspace_of_the_caller(ops):
    lens, H, kvh = [300, 1200, 5], 28, 4
    codes, scales, table = (t.to(DEV) for t in _pool(lens, 256, kvh, 128, 16, seed=30))
    wide = _rows((3, 40, 128), 31).bfloat16().to(DEV)
    q = wide[:, 4:32]
    big = torch.full((3, 36, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = ops.swa_decode_q8_workspace(3, H, 128, DEV)
    if ws is not None:
        ws.fill_(0xFF)                                                       # contents need no initialisation
    out = ops.swa_decode_q8(q, codes[0].view(torch.uint8), codes[1].view(torch.uint8), scales[0], scales[1], table, ln,
                            window_left=256, out=big[:, 8:], workspace=ws)
    _check(out, None, ref.decode(q, codes, scales, table, lens, 256, 128 ** -0.5))
    assert (big[:, :8] == 7.0).all()
    again = ops.swa_decode_q8(q, codes[0], codes[1], scales[0], scales[1], table, ln, window_left=256, workspace=ws)
    assert torch.equal(again, out)


@gpu
def test_attention_refuses_a_workspace_with_gaps_or_too_small(ops):
    codes, scales, table = (t.to(DEV) for t in _pool([40], -1, 1, 128, 16, seed=86))
    q = _rows((1, 7, 128), 87).bfloat16().to(DEV)
    one = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    n = ops.swa_decode_q8_workspace(1, 7, 128, DEV).numel()
    gaps = torch.empty(n, 2, dtype=torch.uint8, device=DEV)[:, 0]
    spread = torch.empty(1, dtype=torch.uint8, device=DEV).expand(1 << 28)
    for ws in (gaps, spread):
        with pytest.raises(ValueError, match="contiguous"):
            ops.swa_decode_q8(q, *codes, *scales, table, one(40), window_left=-1, workspace=ws)
        with pytest.raises(ValueError, match="contiguous"):
            ops.swa_prefill_q8(q, *codes, *scales, table, one(0, 1), one(39), 1, window_left=-1, workspace=ws)
    small = torch.empty(n - 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError):
        ops.swa_decode_q8(q, *codes, *scales, table, one(40), window_left=-1, workspace=small)


@gpu
def test_decode_bad_block_is_reported_and_contained(ops):
    lens = [300, 300, 300]
    codes, scales, table = _pool(lens, -1, 4, 128, 16, seed=32)
    good = table.clone()
    table[1, 3], table[1, 10] = -1, 10 ** 6
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    q = _rows((3, 28, 128), 33).bfloat16().to(DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st = _status()
    out = ops.swa_decode_q8(q, codes[0], codes[1], scales[0], scales[1], table, ln, window_left=-1, status=st)
    assert st.item() == 2 and torch.isfinite(out.float()).all()
    want = ref.decode(q, codes, scales, good.to(DEV), lens, -1, 128 ** -0.5)
    for b in (0, 2):
        _check(out[b:b + 1], None, tuple(t[b:b + 1] for t in want))


@gpu
def test_decode_nan_and_infinity_reach_their_own_rows_only(ops):
    lens = [40, 40, 40]
    codes, scales, table = _pool(lens, -1, 1, 128, 16, seed=34)
    codes.view(torch.uint8)[0, int(table[1, 0]), 3, 0, 5] = 0x7F             # a NaN in a visible key of sequence 1
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    q = _rows((3, 7, 128), 35).bfloat16()
    q[2, 4, 9] = math.inf
    q = q.to(DEV)
    out = ops.swa_decode_q8(q, codes[0], codes[1], scales[0], scales[1], table,
                            torch.tensor(lens, dtype=torch.int32, device=DEV), window_left=-1)
    bad = torch.isnan(out.float()).all(-1).cpu()
    want = torch.zeros(3, 7, dtype=torch.bool)
    want[1], want[2, 4] = True, True
    assert torch.equal(bad, want) and torch.isfinite(out.float()[~bad.to(DEV)]).all()


@gpu
def test_decode_reads_far_into_a_large_pool(ops):
    """Blocks whose byte offset does not fit 32 bits."""
    bs, kvh, nb = 16, 4, 560000                                              # 4.6 GB of K and of V
    codes = torch.empty(2, nb, bs, kvh, 128, dtype=torch.uint8, device=DEV)
    scales = torch.empty(2, nb, kvh, bs, dtype=torch.uint8, device=DEV)
    lens = [50, 200]
    c, s, t = _pool(lens, -1, kvh, 128, bs, seed=36, slack=0)
    far = nb - c.shape[1]
    codes[:, far:], scales[:, far:] = c.view(torch.uint8).to(DEV), s.to(DEV)
    table = torch.where(t >= 0, t + far, t).to(DEV)
    q = _rows((2, 28, 128), 37).bfloat16().to(DEV)
    args = (codes[0], codes[1], scales[0], scales[1], table, torch.tensor(lens, dtype=torch.int32, device=DEV))
    st = _status()
    out = ops.swa_decode_q8(q, *args, window_left=-1, status=st)
    want = ref.decode(q, c.to(DEV), s.to(DEV), t.to(DEV), lens, -1, 128 ** -0.5)
    _check(out, None, want)
    k, _ = ops.kv_gather_q8(*args, 200, status=st)
    assert torch.equal(k[1].double(), ref.window_values(c[0].to(DEV), s[0].to(DEV), t[1].to(DEV), 0, 200).transpose(0, 1))
    new = _rows((1, kvh, 128), 38).bfloat16().to(DEV)
    slot = torch.tensor([nb * bs - 1], device=DEV)
    ops.kv_append_q8(new, new, *args[:4], slot, status=st)
    assert torch.equal(codes[1, nb - 1, bs - 1].cpu(), ref.quantise(new[0])[0]) and st.item() == 0


def _runs(ops, ctx, new, wl, H, kvh, bs, seed, spread=3.0, qmag=1.0, scale=128 ** -0.5):
    lens = [a + b for a, b in zip(ctx, new)]
    codes, scales, table = (t.to(DEV) for t in _pool(lens, wl, kvh, 128, bs, seed, spread, n_new=new))
    T = sum(new)
    q = (qmag * _rows((T + 3, H, 128), seed + 1)).bfloat16().to(DEV)
    out = torch.full((T + 3, H, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    st = _status()
    ops.swa_prefill_q8(q, codes[0], codes[1], scales[0], scales[1], table, start,
                       torch.tensor(ctx, dtype=torch.int32, device=DEV), max(new), window_left=wl, scale=scale, out=out, status=st)
    assert st.item() == 0
    assert (out[T:] == 7.0).all()                                            # rows behind the last sequence stay
    _check(out[:T], None, ref.runs(q[:T], codes, scales, table, ctx, new, wl, scale))


@gpu
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0], [16]), ([0], [17]), ([5], [40]), ([0, 100, 33], [70, 3, 129]),
                                     ([700], [1]), ([0, 9, 200, 64], [5, 0, 1, 64]), ([4000, 1], [2, 300])])
def test_runs_small(ops, ctx, new):
    _runs(ops, ctx, new, 4096, 28, 4, 16, seed=40)


@gpu
@pytest.mark.parametrize("wl", [0, 15, 16, 127, 128, 255, 4096, -1])
def test_runs_windows(ops, wl):
    _runs(ops, [0, 300, 4111], [260, 37, 150], wl, 28, 4, 16, seed=42)


@gpu
@pytest.mark.parametrize("H,kvh,bs", [(7, 1, 16), (14, 2, 32), (32, 4, 64), (4, 4, 16), (16, 2, 128), (3, 1, 48)])
def test_runs_head_layouts_and_block_sizes(ops, H, kvh, bs):
    _runs(ops, [0, 77, 500], [200, 65, 33], 300, H, kvh, bs, seed=44)


@gpu
@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 9])
def test_runs_of_a_few_tokens_on_many_sequences(ops, new):
    _runs(ops, [10, 513, 0, 1000, 64, 2047, 31] * 6, [new] * 42, 700, 28, 4, 16, seed=46)


@gpu
@pytest.mark.parametrize("spread,qmag", [(60.0, 1.0), (0.0, 60.0), (10.0, 1e-3)])
def test_runs_magnitudes(ops, spread, qmag):
    _runs(ops, [500, 3], [40, 300], 350, 28, 4, 16, seed=48, spread=spread, qmag=qmag)


SHORT = ([0, 5, 300, 1500, 31, 2000, 0], [16, 1, 7, 4, 0, 13, 3])            # runs that stream the cache, four queries at a time


@gpu
@pytest.mark.parametrize("wl", [0, 1, 14, 15, 16, 31, 127, 1000, -1])
def test_short_runs_windows(ops, wl):
    _runs(ops, *SHORT, wl, 28, 4, 16, seed=90)


@gpu
@pytest.mark.parametrize("H,kvh,bs", [(7, 1, 16), (14, 2, 32), (32, 4, 64), (4, 4, 16), (16, 2, 128), (3, 1, 48), (2, 2, 16), (8, 1, 16)])
@pytest.mark.parametrize("most", [2, 16])
def test_short_runs_head_layouts_and_block_sizes(ops, H, kvh, bs, most):
    _runs(ops, SHORT[0], [min(n, most) for n in SHORT[1]], 700, H, kvh, bs, seed=92)


@gpu
@pytest.mark.parametrize("spread,qmag,scale", [(60.0, 1.0, 128 ** -0.5), (0.0, 60.0, 128 ** -0.5), (10.0, 1e-3, 128 ** -0.5),
                                               (3.0, 1.0, -0.1), (3.0, 1.0, 0.0), (80.0, 1e-4, 1.0)])
def test_short_runs_magnitudes_and_scales(ops, spread, qmag, scale):
    _runs(ops, *SHORT, 700, 28, 4, 16, seed=94, spread=spread, qmag=qmag, scale=scale)


@gpu
@pytest.mark.parametrize("ctx,new", [([20000], [4]), ([9000, 3, 40000], [11, 16, 5]), ([100] * 350, [12] * 350),
                                     ([130, 0, 4000] * 110, [3, 4, 2] * 110), ([500] * 283, [4] * 283)])
def test_short_runs_cut_into_pieces_and_in_several_launches(ops, ctx, new):
    _runs(ops, ctx, new, -1 if len(ctx) < 4 else 600, 14, 2, 16, seed=96)


@gpu
def test_short_runs_keep_nan_and_bad_blocks_to_their_own_rows(ops):
    ctx, new = [60, 60, 60], [4, 4, 4]
    codes, scales, table = _pool([64, 64, 64], -1, 1, 128, 16, seed=98)
    codes.view(torch.uint8)[0, int(table[1, 3]), 15, 0, 5] = 0x7F            # the newest key of sequence 1: its last query alone
    table[2, 1] = -1
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    q = _rows((12, 7, 128), 99).bfloat16()
    q[2, 4, 9] = math.inf
    st = _status()
    out = ops.swa_prefill_q8(q.to(DEV), codes[0], codes[1], scales[0], scales[1], table,
                             torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=DEV),
                             torch.tensor(ctx, dtype=torch.int32, device=DEV), 4, window_left=-1, status=st)
    bad = torch.isnan(out.float()).all(-1).cpu()
    want = torch.zeros(12, 7, dtype=torch.bool)
    want[2, 4], want[7] = True, True
    assert st.item() == 2 and torch.equal(bad, want) and torch.isfinite(out.float()[~bad.to(DEV)]).all()


@gpu
def test_runs_bad_block_is_reported_and_contained(ops):
    ctx, new = [200, 200], [50, 50]
    codes, scales, table = _pool([250, 250], -1, 4, 128, 16, seed=50)
    good = table.clone().to(DEV)
    table[0, 2] = -1
    codes, scales, table = codes.to(DEV), scales.to(DEV), table.to(DEV)
    q = _rows((100, 28, 128), 51).bfloat16().to(DEV)
    st = _status()
    out = ops.swa_prefill_q8(q, codes[0], codes[1], scales[0], scales[1], table,
                             torch.tensor([0, 50, 100], dtype=torch.int32, device=DEV),
                             torch.tensor(ctx, dtype=torch.int32, device=DEV), 50, window_left=-1, status=st)
    assert st.item() == 2 and torch.isfinite(out.float()).all()
    want = ref.runs(q, codes, scales, good, ctx, new, -1, 128 ** -0.5)
    _check(out[50:], None, tuple(t[50:] for t in want))


# ------------------------------------------------------------------------------------- together, as a serving loop has them
@gpu
def test_a_sequence_written_in_pieces_equals_the_whole_and_decodes_like_its_values(ops):
    """Prompt in two chunks, then token by token (captured into a graph), against one append of everything; the attention
    against the bf16 kernel over the values that the gather returns."""
    B, H, kvh, D, bs, wl, n = 3, 28, 4, 128, 16, 100, 150
    k, v, q = (_rows((B, n, h, D), 60 + i).bfloat16().to(DEV) for i, h in enumerate((kvh, kvh, H)))
    per = -(-n // bs)
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(63)).to(torch.int32).view(B, per).contiguous().to(DEV)
    at = torch.arange(n, device=DEV)
    slots = table.long()[:, at // bs] * bs + at % bs                        # [B, n]
    cache = [ops.kv_cache_q8(B * per, bs, kvh, D, device=DEV) for _ in range(2)]
    st = _status()

    def put(kv, sc, lo, hi):
        ops.kv_append_q8(k[:, lo:hi].reshape(-1, kvh, D), v[:, lo:hi].reshape(-1, kvh, D), kv[0], kv[1], sc[0], sc[1],
                         slots[:, lo:hi].reshape(-1).contiguous(), status=st)
    put(*cache[0], 0, n)
    kv, sc = cache[1]
    put(kv, sc, 0, 90)
    put(kv, sc, 90, 130)
    side = torch.cuda.Stream()
    kt, vt, qt = (torch.zeros(B, h, D, dtype=torch.bfloat16, device=DEV) for h in (kvh, kvh, H))
    slot, lens = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)

    def step():
        ops.kv_append_q8(kt, vt, kv[0], kv[1], sc[0], sc[1], slot, status=st)
        return ops.swa_decode_q8(qt, kv[0], kv[1], sc[0], sc[1], table, lens, window_left=wl, status=st)
    slot.fill_(-1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(130, n):
        kt.copy_(k[:, i]), vt.copy_(v[:, i]), qt.copy_(q[:, i])
        slot.copy_(slots[:, i])
        lens.fill_(i + 1)
        graph.replay()
        _check(out, None, ref.decode(q[:, i], kv, sc, table, [i + 1] * B, wl, D ** -0.5))
    assert st.item() == 0
    assert torch.equal(kv.view(torch.uint8), cache[0][0].view(torch.uint8)) and torch.equal(sc, cache[0][1])
    # the last chunk as a run of queries, on another stream
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        run = ops.swa_prefill_q8(q[:, 130:].reshape(-1, H, D), kv[0], kv[1], sc[0], sc[1], table,
                                 torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=DEV),
                                 torch.full((B,), 130, dtype=torch.int32, device=DEV), 20, window_left=wl, status=st)
    side.synchronize()
    _check(run, None, ref.runs(q[:, 130:].reshape(-1, H, D), kv, sc, table, [130] * B, [20] * B, wl, D ** -0.5))
    kd, vd = ops.kv_gather_q8(kv[0], kv[1], sc[0], sc[1], table, lens, wl + 1, window_left=wl, status=st)
    want, _, err, _ = ref.decode(q[:, n - 1], kv, sc, table, [n] * B, wl, D ** -0.5)
    plain = torch.softmax(torch.einsum("bhgd,bhnd->bhgn", q[:, n - 1].double().view(B, kvh, 7, D), kd.double()) * D ** -0.5, -1)
    assert ((torch.einsum("bhgn,bhnd->bhgd", plain, vd.double()).reshape(B, H, D) - want).abs() <= err + 1e-12).all()
    assert st.item() == 0


# ------------------------------------------------------------------------------------- the framework's surfaces
def _impl(dtype="fp8_e4m3", window=64, H=28, kvh=4):
    from spikingbrain_7b_b200.backend import MetaAttentionImpl
    return MetaAttentionImpl(H, 128, 128 ** -0.5, kvh, None, window, dtype)


def _meta(ctx, new, n_prefill, table, slots, dev):
    from spikingbrain_7b_b200.backend import MetaAttentionMetadata
    lens = [a + b for a, b in zip(ctx, new)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    return MetaAttentionMetadata(
        num_prefills=n_prefill, num_prefill_tokens=sum(new[:n_prefill]), num_decode_tokens=sum(new[n_prefill:]),
        slot_mapping=slots, seq_lens=lens, seq_lens_tensor=i32(lens), max_prefill_seq_len=max(lens[:n_prefill], default=0),
        max_decode_seq_len=max(lens[n_prefill:], default=0), context_lens_tensor=i32(ctx), block_tables=table,
        use_cuda_graph=False, max_query_len=max(new), max_decode_query_len=max(new[n_prefill:], default=1),
        query_start_loc=i32(start), seq_start_loc=i32([sum(lens[:i]) for i in range(len(lens) + 1)]))


def test_backend_takes_the_8_bit_cache_and_refuses_what_it_does_not_have(sb):
    from spikingbrain_7b_b200.backend import MetaAttentionBackend, MetaAttentionImpl
    assert MetaAttentionBackend.get_kv_scale_shape(7, 32, 4) == (2, 7, 4, 32)
    with pytest.raises(ValueError):
        MetaAttentionBackend.get_kv_scale_shape(7, 24, 4)
    for other in ("fp8", "fp8_e5m2", "int8"):
        with pytest.raises(NotImplementedError):
            MetaAttentionImpl(28, 128, 1.0, 4, None, 4097, other)
    impl = _impl()
    q, k = torch.zeros(1, 28, 128).bfloat16(), torch.zeros(1, 4, 128).bfloat16()
    md = _meta([3], [1], 0, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64), "cpu")
    kv, sc = torch.zeros(2, 4, 16, 4, 128, dtype=torch.uint8), torch.zeros(2, 4, 4, 16, dtype=torch.uint8)
    with pytest.raises(ValueError):                                          # codes without exponents
        impl.forward(None, q, k, k, None, None, None, kv, md, output=torch.empty_like(q))
    with pytest.raises(NotImplementedError):                                 # meta tokens
        MetaAttentionImpl(28, 128, 1.0, 4, None, 64, "fp8_e4m3", num_meta_tokens=1).forward(
            None, q, k, k, None, k, k, kv, md, output=torch.empty_like(q), kv_scales=sc)
    with pytest.raises(ValueError):                                          # exponents without codes
        _impl("auto").forward(None, q, k, k, None, None, None, torch.zeros(2, 4, 16, 4, 128).bfloat16(), md,
                              output=torch.empty_like(q), kv_scales=sc)
    from spikingbrain_7b_b200.hf_cache import Cache
    with pytest.raises(NotImplementedError):
        Cache(kv_dtype="int8")


@gpu
@pytest.mark.parametrize("rotary", [False, True])
def test_backend_forward_over_the_8_bit_cache(ops, rotary):
    """Two prompt chunks and two decoding sequences in one call, then a call whose sequences verify several tokens each:
    K/V are written in 8 bits and every output is the attention over the values the cache holds."""
    H, kvh, D, bs, W = 28, 4, 128, 16, 65
    ctx, new = [30, 0, 90, 7], [50, 20, 1, 1]
    impl = _impl(window=W)
    rows, nb = len(ctx), 60
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(80))[:rows * 12].to(torch.int32).view(rows, 12).to(DEV)
    kv, sc = ops.kv_cache_q8(nb, bs, kvh, D, device=DEV)
    cos_sin = ops.build_cos_sin_cache(D, 256, device=DEV)

    def slots_of(ctx, new):
        return torch.cat([table[s].long()[torch.arange(c, c + n, device=DEV) // bs] * bs
                          + torch.arange(c, c + n, device=DEV) % bs for s, (c, n) in enumerate(zip(ctx, new))])
    k0, v0 = (_rows((sum(ctx), kvh, D), 81 + i).bfloat16().to(DEV) for i in range(2))
    ops.kv_append_q8(k0, v0, kv[0], kv[1], sc[0], sc[1], slots_of([0] * rows, ctx))
    for step, (ctx, new, n_prefill) in enumerate([(ctx, new, 2), ([80, 20, 91, 8], [3, 1, 4, 2], 0)]):
        T = sum(new)
        q, k, v = (_rows((T, h, D), 83 + 10 * step + i).bfloat16().to(DEV) for i, h in enumerate((H, kvh, kvh)))
        slots = slots_of(ctx, new)
        kw = {}
        want_kv, want_sc = kv.view(torch.uint8).clone(), sc.clone()
        qr, kr = q.clone(), k.clone()
        if rotary:
            pos = torch.cat([torch.arange(c, c + n, device=DEV) for c, n in zip(ctx, new)])
            kw = {"positions": pos, "cos_sin_cache": cos_sin}
            ops.rope_kv_append_q8(qr, kr, v, want_kv[0], want_kv[1], want_sc[0], want_sc[1], slots, pos, cos_sin, key_in_place=True)
        else:
            ops.kv_append_q8(kr, v, want_kv[0], want_kv[1], want_sc[0], want_sc[1], slots)
        out = torch.empty(T, H * D, dtype=torch.bfloat16, device=DEV)
        impl.forward(None, q, k, v, None, None, None, kv, _meta(ctx, new, n_prefill, table, slots, DEV), output=out, kv_scales=sc, **kw)
        assert impl.status() == 0
        assert torch.equal(kv.view(torch.uint8), want_kv) and torch.equal(sc, want_sc)
        assert torch.equal(q, qr) and torch.equal(k, kr)
        _check(out.view(T, H, D), None, ref.runs(qr, kv, sc, table, ctx, new, W - 1, D ** -0.5))


@gpu
def test_backend_block_moves_take_codes_and_exponents(ops):
    from spikingbrain_7b_b200.backend import MetaAttentionBackend
    codes, scales, table = _pool([100], -1, 2, 128, 16, seed=90)
    kv, sc = codes.to(DEV), scales.to(DEV)
    want = (kv.view(torch.uint8).clone(), sc.clone())
    pairs = torch.tensor([[int(table[0, 0]), 8], [int(table[0, 1]), 9]])
    MetaAttentionBackend.copy_blocks([kv, sc], pairs)
    other = (torch.zeros_like(kv.view(torch.uint8)).view(kv.dtype), torch.zeros_like(sc))
    for a, b in zip((kv, sc), other):
        MetaAttentionBackend.swap_blocks(a, b, pairs)
    for src, dst in pairs.tolist():
        assert torch.equal(kv.view(torch.uint8)[:, dst], want[0][:, src]) and torch.equal(sc[:, dst], want[1][:, src])
        assert torch.equal(other[0].view(torch.uint8)[:, dst], want[0][:, src]) and torch.equal(other[1][:, dst], want[1][:, src])


@gpu
@pytest.mark.parametrize("window,dtype,D", [(24, torch.bfloat16, 128), (24, torch.float32, 64), (None, torch.bfloat16, 128)])
def test_hf_cache_in_8_bits_holds_the_quantised_window(ops, window, dtype, D):
    """The stream of the reference class with every token replaced by what the 8-bit format makes of it, also across the
    growth of an unbounded layer; decode against attention over exactly those values."""
    from spikingbrain_7b_b200.hf_cache import Cache
    B, kvh, H = 2, 4, 28
    cache = Cache(kv_dtype="fp8_e4m3", unbounded_capacity=40)
    oracle = ref_ops.RefWindowCache()
    for step, n in enumerate([20, 4] + [1] * 60):
        if step == 1 and window is not None:
            n = window - 20
        k, v = (_rows((B, kvh, n, D), 100 + 2 * step + i).to(dtype) for i in range(2))
        st = cache.update(attn_state=(k.to(DEV), v.to(DEV)), layer_idx=0, offset=n, cache_kwargs={"window_size": window})
        kq, vq = (ref.values(*ref.quantise(x)).to(dtype) for x in (k, v))
        want = oracle.update(attn_state=(kq, vq), layer_idx=0, offset=n, cache_kwargs={"window_size": window})["attn_state"]
        for a, b in zip(st["attn_state"], want):
            assert a.dtype == dtype and torch.equal(a.cpu(), b)
        if D == 128 and n == 1 and step % 9 == 0:
            q = _rows((B, H, D), 300 + step).bfloat16().to(DEV)
            out = cache.swa_decode(q, 0)
            for b in range(B):
                kk, vv = (t[b].transpose(0, 1).to(DEV) for t in want)
                seen = torch.ones(1, kk.shape[0], dtype=torch.bool, device=DEV)
                _check(out[b:b + 1], None, ref.attend(q[b:b + 1], kk, vv, seen, D ** -0.5))
    assert cache.status() == 0
    legacy = cache.to_legacy_cache()
    again = Cache.from_legacy_cache(legacy, seen_tokens=cache.get_seq_length(), kv_dtype="fp8_e4m3")
    k, v = (_rows((B, kvh, 1, D), 400 + i).to(dtype) for i in range(2))
    got = again.update(attn_state=(k.to(DEV), v.to(DEV)), layer_idx=0, offset=1, cache_kwargs={"window_size": window})["attn_state"]
    kq = ref.values(*ref.quantise(k)).to(dtype)
    old = legacy[0]["attn_state"][0].cpu()
    keep = old if window is None else old[..., -(window - 1):, :]
    assert torch.equal(got[0].cpu(), torch.cat([keep, kq], -2))              # quantising values again changes nothing


@gpu
def test_hf_cache_in_8_bits_with_rotary(ops):
    from spikingbrain_7b_b200.hf_cache import Cache
    B, kvh, H, D, W = 2, 4, 28, 128, 20
    table = ops.build_cos_sin_cache(D, 512, device=DEV)
    cache = Cache(kv_dtype="fp8_e4m3")
    for n, p0 in ((33, 0), (1, 33), (1, 34)):                                # a prompt longer than the window, then tokens
        q, k, v = (_rows((B, h, n, D), 500 + p0 + i).bfloat16().to(DEV) for i, h in enumerate((H, kvh, kvh)))
        pos = torch.arange(p0, p0 + n, device=DEV).unsqueeze(0)
        c, s = table.double()[pos[0], :64], table.double()[pos[0], 64:]
        turn = lambda x: torch.cat([x.double()[..., :64] * c - x.double()[..., 64:] * s,
                                    x.double()[..., 64:] * c + x.double()[..., :64] * s], -1)
        want_q, want_k = turn(q), turn(k)
        got = cache.update_rotary(q, k, v, pos, table, 0, window_size=W)
        assert ((got.double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -21 * q.double().abs().amax()).all()
        m = min(n, W)
        newest = cache[0]["attn_state"][0][:, :, -m:].double()
        want_k = want_k[:, :, -m:]
        # nearest code: half a step of the value, or of the smallest codes of its row (2^-10 of a 448th of the row's largest)
        bound = torch.maximum(want_k.abs() * 2.0 ** -4, want_k.abs().amax(-1, keepdim=True) * 2.0 ** -17) * (1 + 2.0 ** -10)
        assert ((newest - want_k).abs() <= bound).all()
    assert cache.status() == 0
