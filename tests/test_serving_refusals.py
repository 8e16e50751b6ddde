"""More of the host side of the 8-bit cache and row sampling entry points."""
import pytest

from test_serving_cpu import refused


def test_wait_limits_out_of_range_are_refused(qtts):
    refused(qtts, lambda: qtts.kv8_wait_limit(-1))
    refused(qtts, lambda: qtts.kv8_wait_limit(2_000_000_001))
    qtts.kv8_wait_limit(0)
    qtts.kv8_wait_limit()


def test_the_timeout_bit_matches_the_header(qtts):
    assert f"#define QTTS_KV8_TIMEOUT {qtts.KV8_TIMEOUT} " in open(qtts.HEADER).read()
