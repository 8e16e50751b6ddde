"""Corners of the 8-bit cache operators on the GPU: what the documentation
allows and ordinary data does not reach."""
import numpy as np
import pytest

import serving_ref as R
from conftest import has_gpu
from test_gpu_kv8 import Pool, check_attention, dev, host, rows_of, run_append, tables

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


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hd,length", [(128, 30000), (64, 32001)])
def test_long_f32_tiles_sum_their_weights_in_full(qtts, hd, length, sign):
    # So many units that no cluster shares the positions: a slot adds up the
    # weights of the whole cache, page by page (a negative scale takes the path
    # of any tile, otherwise used for masked ones).  The bound of
    # test_long_f32_sums_are_rounded, here for every row and head, as an error of
    # the weights' sum is common to all of a row: the weights are off by 2^-21
    # with random sign, rounded sums of 250 tiles by 2^-20 at most, and the sum
    # of the weights, compensated, by 2^-23.  Plain sums of n weights are off by
    # about sqrt(n) 2^-25 and up to n 2^-24: 5e-6 for 30000.
    rng = np.random.default_rng(length)
    kvh, n_seqs, rows = 8, 10, 128
    p = Pool(qtts, rng, 1, (length + 15) // 16, kvh, hd)
    table = p.d_table.expand(n_seqs, -1).contiguous()
    cache = qtts.Kv8Cache(p.d_codes.data_ptr(), p.d_scales.data_ptr(), table.data_ptr(), p.codes.shape[0], n_seqs,
                          table.shape[1], kvh, hd)
    seq, pos = rows_of([(s, length - rows, rows) for s in range(n_seqs)])
    q = dev((rng.standard_normal((len(seq), kvh * hd)) * 0.3).astype(np.float32))
    out, lse = torch.empty_like(q), torch.empty(len(seq), kvh, device="cuda")
    t = dev(seq), dev(pos)
    scale = sign * hd ** -0.5
    qtts.kv8_attention_dev(cache, q.data_ptr(), out.data_ptr(), t[0].data_ptr(), t[1].data_ptr(), len(seq), kvh,
                           scale=scale, max_rows=rows, max_len=length, lse_ptr=lse.data_ptr())
    torch.cuda.synchronize()
    at = dev(p.table[0].astype(np.int64))
    kv = p.d_codes[at, 0].double() * p.d_scales[at, 0].double()[..., None, None]
    kv = kv.permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, hd)[:, :, :length]
    worst = 0.0
    for h in range(kvh):
        a = q[:, h * hd:(h + 1) * hd].double() @ kv[0, h].T * scale
        a.masked_fill_(torch.arange(length, device="cuda")[None] > t[1][:, None], -float("inf"))
        want = torch.softmax(a, -1) @ kv[1, h]
        err = (out[:, h * hd:(h + 1) * hd].double() - want).norm(dim=-1) / want.norm(dim=-1)
        worst = max(worst, err.max().item())
        # log2 of the sum, its product with ln 2 and the result, each rounded (values up to 16)
        assert float((lse[:, h].double() - torch.logsumexp(a, -1)).abs().max()) <= 2.0 ** -19 + 16 * 3 * 2.0 ** -24
    print("worst row", worst)
    assert worst <= 2.0 ** -19


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", ["whole", "split"])
def test_a_wait_that_runs_out_marks_its_rows(qtts, dtype, shape):
    # A wait that nothing ends, with no time given: every CTA gives up, the call
    # ends, the rows are NaN (padding rows stay), the flag says why, and the next
    # call is right.
    rng = np.random.default_rng(31)
    # (shapes that tiles take; single tokens and few rows have nothing to wait for)
    n_seqs, rows, length, kvh, hd = (8, 100, 200, 8, 64) if shape == "whole" else (1, 400, 3000, 2, 128)
    heads = 2 * kvh
    p = Pool(qtts, rng, n_seqs, (length + 15) // 16, kvh, hd)
    seq, pos = rows_of([(s, length - rows, rows) for s in range(n_seqs)] + [(-1, 0, 3)])
    n = len(seq)
    q = dev(rng.standard_normal((n, heads * hd)).astype(np.float32), dtype)
    t = dev(seq), dev(pos)
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call(out, lse):
        qtts.kv8_attention_dev(p.cache, q.data_ptr(), out.data_ptr(), t[0].data_ptr(), t[1].data_ptr(), n, heads,
                               dtype=dtype, max_rows=rows, lse_ptr=lse.data_ptr(), flags_ptr=flags.data_ptr())

    want, wlse = torch.full_like(q, 5.0), torch.full((n, heads), 5.0, device="cuda")
    call(want, wlse)
    torch.cuda.synchronize()
    assert flags.item() == 0 and bool(torch.isfinite(want).all())
    for again in range(2):
        out, lse = torch.full_like(q, 5.0), torch.full((n, heads), 5.0, device="cuda")
        qtts.kv8_wait_limit(0)
        try:
            call(out, lse)
        finally:
            qtts.kv8_wait_limit()
        torch.cuda.synchronize()
        assert flags.item() == qtts.KV8_TIMEOUT
        assert bool(out[:n - 3].isnan().all()) and bool(lse[:n - 3].isnan().all())
        assert bool((out[n - 3:] == 5.0).all()) and bool((lse[n - 3:] == 5.0).all())
        flags.zero_()
        out, lse = torch.full_like(q, 5.0), torch.full((n, heads), 5.0, device="cuda")
        call(out, lse)
        torch.cuda.synchronize()
        assert flags.item() == 0 and torch.equal(out, want) and torch.equal(lse, wlse)


def by_row_and_head(p, q, heads, seq, pos, scale, window):
    """64-bit attention [n][heads][hd] and, for its error, of every row and head:
    the sums of weight * |v|, the largest weight * V scale, the largest
    scale * sum |q k|, and the number of positions seen."""
    kvh, hd, cap = p.codes.shape[2], p.hd, p.table.shape[1] * 16
    n = len(seq)
    want, mass = np.zeros((2, n, heads, hd))
    heavy, most = np.zeros((2, n, heads))
    seen = np.zeros(n)
    for r in range(n):
        if pos[r] < 0:
            continue
        lo = max(0, pos[r] + 1 - window) if window else 0
        at = np.arange(lo, min(int(pos[r]), cap - 1) + 1)
        page = p.table[seq[r], at // 16]
        seen[r] = len(at)
        for h in range(heads):
            k, v = (p.codes[page, i, h * kvh // heads, at % 16].astype(np.float64) *
                    p.scales[page, i, h * kvh // heads, None].astype(np.float64) for i in (0, 1))
            x = q[r, h * hd:(h + 1) * hd].astype(np.float64)
            a = k @ x * scale
            w = np.exp(a - a.max())
            w /= w.sum()
            want[r, h], mass[r, h] = w @ v, w @ np.abs(v)
            heavy[r, h] = (w * np.abs(p.scales[page, 1, h * kvh // heads].astype(np.float64))).max()
            most[r, h] = abs(scale) * (np.abs(k) @ np.abs(x)).max()
    return want, mass, heavy, most, seen


@pytest.mark.parametrize("rows,max_rows,n_seqs,kvh,hd", [(1, 1, 8, 8, 64), (3, 3, 8, 2, 128), (100, 100, 8, 8, 64),
                                                        (100, 1, 2, 2, 64), (60, 60, 12, 8, 128)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 60])
def test_scales_far_apart_row_by_row(qtts, rows, max_rows, n_seqs, kvh, hd, dtype, window):
    # V scales of 1e-9 .. 1e9 in an order that grows, falls or jumps, so that the
    # running exponent moves both ways; each row and head against its own bound
    rng = np.random.default_rng(rows + hd + window)
    per = 20
    p = Pool(qtts, rng, n_seqs, per, kvh, hd)
    power = rng.integers(-9, 10, (len(p.scales), kvh)).astype(np.float64)
    for s in range(n_seqs):
        if s % 4 == 1:
            power[p.table[s]] = np.linspace(-9, 9, per)[:, None]
        elif s % 4 == 2:
            power[p.table[s]] = np.linspace(9, -9, per)[:, None]
    p.scales[:, 1] *= (10.0 ** power).astype(np.float32)
    p.scales[p.table[0, 2], 1] = 0.0
    p.scales[p.table[0, 3], 0] = 0.0
    p.scales[p.table[1, :5], 1] = 0.0
    p.d_scales[:, 0] = dev(p.scales)
    heads = 2 * kvh
    top = 203 if dtype != "f16" else 150
    seq, pos = rows_of([(s, top - 11 * s if rows == 1 else top, rows) for s in range(n_seqs)])
    if dtype == "f16":  # results that f16 holds
        p.scales[:, 1] = np.clip(p.scales[:, 1], 0, 1)
        p.d_scales[:, 0] = dev(p.scales)
    n = len(seq)
    q = dev(rng.standard_normal((n, heads * hd)).astype(np.float32), dtype)
    out = torch.full_like(q, 5.0)
    t = dev(seq), dev(pos)
    qtts.kv8_attention_dev(p.cache, q.data_ptr(), out.data_ptr(), t[0].data_ptr(), t[1].data_ptr(), n, heads, dtype=dtype,
                           window=window, scale=hd ** -0.5, max_rows=max_rows)
    torch.cuda.synchronize()
    want, mass, heavy, most, seen = by_row_and_head(p, host(q), heads, seq, pos, hd ** -0.5, window)
    # As in check_attention: scores off by d, weights by twice that, 2^-20 for exp2
    # and the pair, 2^-11 where they are f16; sums by 2^-23 a step of 16 positions
    # and 32 for joins; all of weight * |v|.  A pair's lo part is rounded to 2^-25
    # of the row's largest weight * V scale, for a code of up to 127 at every position.
    d = most * (hd / 16 + 8) * 2.0 ** -23
    weights = 2.0 ** -11 if dtype != "f32" and max_rows > 1 else 0.0
    rel = 2 * d + weights + 2.0 ** -20 + ((seen[:, None] + 128) / 16 + 32) * 2.0 ** -23
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    tol = mass * rel[..., None] + (heavy * seen[:, None] * 127 * 2.0 ** -25)[..., None] + half * np.abs(want)
    if dtype == "f16":
        tol = tol + 2.0 ** -25  # its subnormals
    got = host(out).reshape(n, heads, hd).astype(np.float64)
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:3], (np.abs(got - want) / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("heads,kvh", [(300, 1), (39, 3)])
@pytest.mark.parametrize("max_rows", [1, 90])
def test_many_heads_a_cache_head(qtts, heads, kvh, max_rows):
    # more query heads than a tile has slots, and counts that its chunks do not divide
    rng = np.random.default_rng(heads)
    p = Pool(qtts, rng, 2, 8, kvh, 64)
    seq, pos = rows_of([(0, 5, 90), (-1, 0, 1), (1, 100, 20)])
    for dtype in ("f32", "bf16"):
        check_attention(qtts, p, rng, seq, pos, heads, dtype, max_rows=max_rows)


@pytest.mark.parametrize("rows", [1, 150])
def test_hints_and_windows_at_their_ends(qtts, rows):
    # results do not depend on max_rows and max_len, and a window may be any size;
    # positions and sequences far outside are flagged, far below nothing
    rng = np.random.default_rng(rows)
    p = Pool(qtts, rng, 4, 30, 4, 128)
    seq, pos = rows_of([(s, 479 - rows, rows) for s in range(4)])
    q = rng.standard_normal((len(seq), 8 * 128))
    for max_rows in (0, 1, 7, 2 ** 31 - 1):
        for max_len in (0, 1, 2 ** 31 - 1):
            for window in (0, 33, 2 ** 31 - 1):
                check_attention(qtts, p, rng, seq, pos, 8, "f32", q=q, max_rows=max_rows, max_len=max_len, window=window)
    pos[0] = -2 ** 31
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    for max_rows in (1, 150):
        check_attention(qtts, p, rng, seq, pos, 8, "f32", q=q, max_rows=max_rows, window=20, flags=flags)
        assert flags.item() == 0
        far = pos.copy()
        far[-1] = 2 ** 31 - 1
        check_attention(qtts, p, rng, seq, far, 8, "f32", q=q, max_rows=max_rows, flags=flags)
        assert flags.item() == qtts.KV8_BAD_ROW
        flags.zero_()


@pytest.mark.parametrize("n_seqs", [1, 700])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_turned_in_place(qtts, dtype, n_seqs):
    # q_out may be q; an odd number of rows, as a prompt's warps take two each, and
    # the same rows in a pool of many sequences
    rng = np.random.default_rng(n_seqs)
    hd, kvh, heads = 64, 2, 6
    p = Pool(qtts, rng, n_seqs, 4, kvh, hd)
    seq, pos = rows_of([(0, 1, 61), (-1, 0, 2)])
    n = len(seq)
    cos, sin = tables(64, hd)
    gq = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float16)
    dc, ds, dgq, dseq, dpos = dev(cos), dev(sin), dev(gq), dev(seq), dev(pos)
    x = dev(rng.standard_normal((n, (heads + 2 * kvh) * hd)).astype(np.float32), dtype)
    before = host(x)
    ld, b, size = x.stride(0), x.data_ptr(), x.element_size()
    qtts.kv8_append_dev(p.cache, b + heads * hd * size, b + (heads + kvh) * hd * size, dseq.data_ptr(), dpos.data_ptr(), n,
                        dtype=dtype, q_ptr=b, q_out_ptr=b, heads=heads, q_norm_ptr=dgq.data_ptr(), cos_ptr=dc.data_ptr(),
                        sin_ptr=ds.data_ptr(), rope_rows=64, ldk=ld, ldv=ld, ldq=ld, ldqo=ld)
    torch.cuda.synchronize()
    want = before.copy()
    for r in range(n):
        if seq[r] >= 0:
            want[r, :heads * hd] = R.norm_rotate(before[r, :heads * hd].reshape(heads, hd), gq, cos[pos[r]], sin[pos[r]]).reshape(-1)
    assert torch.equal(x, dev(want, dtype))
    k, v = before[:, heads * hd:(heads + kvh) * hd], before[:, (heads + kvh) * hd:]
    R.append(p.codes, p.scales, p.table, k, v, seq, pos, None, cos, sin)
    codes, scales = p.got()
    assert np.array_equal(codes, p.codes) and np.array_equal(scales, p.scales)


@pytest.mark.parametrize("n_seqs", [1, 160])
def test_long_f32_tokens_row_by_row(qtts, n_seqs):
    # the bound of test_long_f32_tiles_sum_their_weights_in_full for single tokens:
    # one sequence whose pages a cluster shares, and so many that a CTA has them alone
    rng = np.random.default_rng(n_seqs)
    kvh, hd, length = 8, 128, 32003
    p = Pool(qtts, rng, 1, (length + 15) // 16, kvh, hd)
    table = p.d_table.expand(n_seqs, -1).contiguous()
    cache = qtts.Kv8Cache(p.d_codes.data_ptr(), p.d_scales.data_ptr(), table.data_ptr(), p.codes.shape[0], n_seqs,
                          table.shape[1], kvh, hd)
    seq, pos = np.arange(n_seqs, dtype=np.int32), (length - 1 - np.arange(n_seqs)).astype(np.int32)
    q = dev((rng.standard_normal((n_seqs, 2 * kvh * hd)) * 0.3).astype(np.float32))
    out, lse = torch.empty_like(q), torch.empty(n_seqs, 2 * kvh, device="cuda")
    t = dev(seq), dev(pos)
    qtts.kv8_attention_dev(cache, q.data_ptr(), out.data_ptr(), t[0].data_ptr(), t[1].data_ptr(), n_seqs, 2 * kvh,
                           max_len=length, lse_ptr=lse.data_ptr())
    torch.cuda.synchronize()
    at = dev(p.table[0].astype(np.int64))
    kv = p.d_codes[at, 0].double() * p.d_scales[at, 0].double()[..., None, None]
    kv = kv.permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, hd)[:, :, :length]
    for h in range(2 * kvh):
        a = q[:, h * hd:(h + 1) * hd].double() @ kv[0, h // 2].T * hd ** -0.5
        a.masked_fill_(torch.arange(length, device="cuda")[None] > t[1][:, None], -float("inf"))
        want = torch.softmax(a, -1) @ kv[1, h // 2]
        err = (out[:, h * hd:(h + 1) * hd].double() - want).norm(dim=-1) / want.norm(dim=-1)
        assert err.max().item() <= 2.0 ** -19, h
        assert float((lse[:, h].double() - torch.logsumexp(a, -1)).abs().max()) <= 2.0 ** -19 + 16 * 3 * 2.0 ** -24
