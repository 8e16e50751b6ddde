"""More of the host side of the 8-bit cache and row sampling entry points."""
import pytest

from test_serving_cpu import X, append, attend, cache, refused


def test_wait_limits_out_of_range_are_refused(qtts):
    refused(qtts, lambda: qtts.kv8_wait_limit(-1))
    refused(qtts, lambda: qtts.kv8_wait_limit(2_000_000_001))
    qtts.kv8_wait_limit(0)
    qtts.kv8_wait_limit()


def test_the_timeout_bit_matches_the_header(qtts):
    assert f"#define QTTS_KV8_TIMEOUT {qtts.KV8_TIMEOUT} " in open(qtts.HEADER).read()


@pytest.mark.parametrize("off", [1, 2])
def test_misaligned_small_arrays_are_refused(qtts, off):
    # a kernel that follows such a pointer faults
    p = X + off
    for kw in (dict(seq=p), dict(pos=p), dict(rope_pos_ptr=p, cos_ptr=X, sin_ptr=X, rope_rows=4), dict(flags_ptr=p)):
        refused(qtts, lambda: append(qtts, cache(qtts), **kw))
    for kw in (dict(seq=p), dict(pos=p), dict(lse_ptr=p), dict(flags_ptr=p)):
        refused(qtts, lambda: attend(qtts, cache(qtts), **kw))
    names = ("temperature_ptr", "top_k_ptr", "top_p_ptr", "min_p_ptr", "kept_ptr", "logprob_ptr")
    for kw in [dict(u=p), dict(token=p)] + [{n: p} for n in names]:
        a = dict(u=X, token=X)
        a.update({k: kw.pop(k) for k in list(kw) if k in a})
        refused(qtts, lambda: qtts.sample_rows_dev(X, 2, 8, a["u"], a["token"], **kw))
