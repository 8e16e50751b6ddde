"""Host side of the 8-bit cache and row sampling entry points: every refusal is
made before the GPU is touched, and the restatements used as their oracle hold
the documented bounds."""
import ctypes as C

import numpy as np
import pytest

import serving_ref as R

X = 1 << 20  # a nonzero, aligned number in a pointer's place: refused calls never follow it


def cache(qtts, **kw):
    a = dict(codes=X, scales=X, table=X, n_pages=4, n_seqs=2, per_seq=2, kvh=2, hd=64, ps=0, ss=0)
    a.update(kw)
    return qtts.Kv8Cache(a["codes"], a["scales"], a["table"], a["n_pages"], a["n_seqs"], a["per_seq"], a["kvh"],
                         a["hd"], a["ps"], a["ss"])


def append(qtts, c, **kw):
    a = dict(k=X, v=X, seq=X, pos=X, n=3)
    a.update({k: kw.pop(k) for k in list(kw) if k in a})
    qtts.kv8_append_dev(c, a["k"], a["v"], a["seq"], a["pos"], a["n"], **kw)


def attend(qtts, c, **kw):
    a = dict(q=X, out=X, seq=X, pos=X, n=3, heads=4)
    a.update({k: kw.pop(k) for k in list(kw) if k in a})
    qtts.kv8_attention_dev(c, a["q"], a["out"], a["seq"], a["pos"], a["n"], a["heads"], **kw)


def refused(qtts, f, code=None):
    with pytest.raises(qtts.QttsError) as e:
        f()
    assert e.value.code == (qtts.ERR_BADARG if code is None else code), e.value


BAD_CACHES = [dict(codes=0), dict(scales=0), dict(table=0), dict(hd=96), dict(kvh=0), dict(kvh=4096), dict(n_pages=0),
              dict(n_seqs=0), dict(per_seq=0), dict(per_seq=1 << 28), dict(ps=4080), dict(ps=8200), dict(ss=3),
              dict(codes=X + 4), dict(scales=X + 2)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(qtts, kw):
    c = cache(qtts, **kw)
    refused(qtts, lambda: append(qtts, c))
    refused(qtts, lambda: attend(qtts, c))


@pytest.mark.parametrize("kw", [dict(k=0), dict(v=0), dict(seq=0), dict(pos=0), dict(n=-1), dict(dtype="e4m3"),
                                dict(ldk=124), dict(ldv=130), dict(k=X + 4), dict(q_ptr=X), dict(q_out_ptr=X, heads=4),
                                dict(q_ptr=X, q_out_ptr=X), dict(q_ptr=X, q_out_ptr=X, heads=4, ldq=255),
                                dict(q_ptr=X + 8, q_out_ptr=X, heads=4), dict(cos_ptr=X), dict(sin_ptr=X, rope_rows=4),
                                dict(cos_ptr=X, sin_ptr=X), dict(cos_ptr=X + 4, sin_ptr=X, rope_rows=4),
                                dict(k_norm_ptr=X + 2)])
def test_bad_appends_are_refused(qtts, kw):
    refused(qtts, lambda: append(qtts, cache(qtts), **kw))


@pytest.mark.parametrize("kw", [dict(q=0), dict(out=0), dict(seq=0), dict(pos=0), dict(n=-1), dict(heads=0),
                                dict(heads=3), dict(heads=32768), dict(dtype="f64"), dict(window=-1),
                                dict(max_rows=-1), dict(max_len=-2), dict(ldq=252), dict(ldo=258), dict(q=X + 8),
                                dict(out=X + 2, dtype="bf16")])
def test_bad_attentions_are_refused(qtts, kw):
    refused(qtts, lambda: attend(qtts, cache(qtts), **kw))


def test_too_many_rows_are_refused(qtts):
    refused(qtts, lambda: attend(qtts, cache(qtts), n=1 << 30), qtts.ERR_RANGE)


def test_no_rows_is_no_work(qtts):
    append(qtts, cache(qtts), k=0, v=0, seq=0, pos=0, n=0)
    attend(qtts, cache(qtts), q=0, out=0, seq=0, pos=0, n=0)
    qtts.sample_rows_dev(0, 0, 5, 0, 0)


def test_null_cache_is_refused(qtts):
    rc = qtts.lib.qtts_kv8_append_dev(None, X, 128, X, 128, None, 0, None, 0, 0, 0, None, None, None, None, 0, X, X,
                                      None, 1, None, None)
    assert rc == qtts.ERR_BADARG and b"null" in qtts.lib.qtts_last_error()
    rc = qtts.lib.qtts_kv8_attention_dev(None, X, 128, 2, 0, 1.0, 0, X, X, 1, 0, 0, X, 128, None, None, None)
    assert rc == qtts.ERR_BADARG


@pytest.mark.parametrize("a,code", [(dict(n=-1), None), (dict(V=0), None), (dict(ld=4), None), (dict(logits=0), None),
                                    (dict(u=0), None), (dict(token=0), None), (dict(dtype="int8"), None),
                                    (dict(logits=X + 1), None), (dict(V=262145), "range")])
def test_bad_samples_are_refused(qtts, a, code):
    b = dict(logits=X, n=2, V=8, u=X, token=X, ld=0, dtype="f32")
    b.update(a)
    refused(qtts, lambda: qtts.sample_rows_dev(b["logits"], b["n"], b["V"], b["u"], b["token"], dtype=b["dtype"],
                                               ld=b["ld"]), qtts.ERR_RANGE if code else None)


def test_the_cache_struct_matches_the_header(qtts):
    assert C.sizeof(qtts.Kv8CacheDesc) == 3 * 8 + 5 * 4 + 4 + 2 * 8
    text = open(qtts.HEADER).read()
    for name, value in [("QTTS_KV8_BAD_ROW", qtts.KV8_BAD_ROW), ("QTTS_KV8_BAD_PAGE", qtts.KV8_BAD_PAGE),
                        ("QTTS_KV8_ROPE_RANGE", qtts.KV8_ROPE_RANGE), ("QTTS_F32", 0), ("QTTS_F16", 1),
                        ("QTTS_BF16", 2), ("QTTS_SAMPLE_ROWS_MAX_V", qtts.SAMPLE_ROWS_MAX_V)]:
        assert f"#define {name} {value}" in text


@pytest.mark.parametrize("step", [1, 3, 16])
@pytest.mark.parametrize("growth", [1.0, 1.02, 1.3])
def test_requantised_blocks_stay_within_two_and_a_half_steps(step, growth):
    # the documented bound, on tokens whose size grows so that blocks are
    # rounded again and again: half a step for a block written at once, and
    # 1/2 (1 + 1/1.25 + ...) = 2.5 final steps for one that grows
    rng = np.random.default_rng(int(10 * growth) + step)
    hd, n = 64, 48
    codes, scales = np.zeros((3, 2, 1, 16, hd), np.int8), np.zeros((3, 2, 1), np.float32)
    table = np.array([[2, 0, 1]])
    k = (rng.standard_normal((n, hd)) * growth ** np.arange(n)[:, None]).astype(np.float32)
    v = rng.standard_normal((n, hd)).astype(np.float32)
    for a in range(0, n, step):
        b = slice(a, min(n, a + step))
        R.append(codes, scales, table, k[b], v[b], np.zeros(n, int)[b], np.arange(n)[b])
    got = (codes.astype(np.float64) * scales[..., None, None])[table[0]].transpose(1, 0, 2, 3, 4).reshape(2, n, hd)
    unit = np.repeat(scales[table[0], :, 0].T, 16, axis=1)[..., None]
    bound = (0.5 if step == 16 else 2.5) * unit * (1 + 1e-5)
    assert np.all(np.abs(got - np.stack([k, v])) <= bound)
