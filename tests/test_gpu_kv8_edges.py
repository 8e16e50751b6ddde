"""Corners of the 8-bit cache operators on the GPU: what the documentation
allows and ordinary data does not reach."""
import numpy as np
import pytest

import serving_ref as R
from conftest import has_gpu
from test_gpu_kv8 import Pool, dev, host, rows_of, run_append, tables

pytestmark = pytest.mark.gpu
if has_gpu():
    import torch


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("parts", [[(0, 0, 1), (1, 5, 1)], [(0, 3, 40), (1, 0, 2)]], ids=["tokens", "chunks"])
def test_a_key_without_angles_keeps_its_infinities_and_their_partners(qtts, hd, norm, parts):
    # rows whose rotation positions lie outside the tables are stored unrotated:
    # an element is itself even if the one half a head away is infinite or NaN
    rng = np.random.default_rng(hd)
    p = Pool(qtts, rng, 3 if len(parts) else 1, 3, 2, hd)
    seq, pos = rows_of(parts)
    n = len(seq)
    k, v = rng.standard_normal((2, n, 2 * hd)).astype(np.float32)
    rope = pos.astype(np.int32).copy()
    rope[::2] = np.where(np.arange(len(rope[::2])) % 2, -1, 48)  # every second row has no angles
    if norm:  # finite, but the mean of its squares is not: the row becomes zeros
        k[::2, 3] = 3e38
    else:
        k[::2, 3] = np.inf
        k[::2, hd + hd // 2 + 7] = -np.inf
        k[::4, 11] = np.nan
    k[::2, hd // 2 + 3] = 50.0  # the largest of its block, and the partner of the first
    g = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float16)
    cos, sin = tables(48, hd)
    dc, ds, dr, dg = dev(cos), dev(sin), dev(rope), dev(g)
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    run_append(qtts, p, k, v, seq, pos, cos_ptr=dc.data_ptr(), sin_ptr=ds.data_ptr(), rope_rows=48,
               rope_pos_ptr=dr.data_ptr(), k_norm_ptr=dg.data_ptr() if norm else 0, flags_ptr=flags.data_ptr())
    with np.errstate(invalid="ignore", over="ignore"):
        R.append(p.codes, p.scales, p.table, k, v, seq, pos, g if norm else None, cos, sin, rope)
    codes, scales = p.got()
    assert np.array_equal(scales, p.scales)
    assert np.array_equal(codes, p.codes)
    assert flags.item() == qtts.KV8_ROPE_RANGE
