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
