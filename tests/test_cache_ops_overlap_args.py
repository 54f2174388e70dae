"""Calls of the cache operators whose outputs overlap another argument are refused, before the device is touched."""
import itertools

import pytest

from swiftlm_b200 import _lib

from .test_cache_attention_args import call

STEP = 1 << 28                       # every argument has a range of its own, larger than it needs
NAMES = "q k v page_table q_len kv_len out lse mass ws kv_len_out mass_out kept".split()
PAGED = dict(page_tokens=16, max_pages=8, num_pages=40, N=100, B=5, T=20)         # the smallest argument: 20 bytes
USED = {"decode": "q k v page_table kv_len out lse mass ws".split(), "prompt": "q k v page_table q_len kv_len out lse ws".split(),
        "mass": "q k page_table q_len kv_len lse mass ws".split(),
        "evict": "k v page_table kv_len mass ws kv_len_out mass_out kept".split()}
WRITTEN = {"decode": {"out", "lse", "mass", "ws"}, "prompt": {"out", "lse", "ws"}, "mass": {"mass", "ws"},
           "evict": {"k", "v", "ws", "kv_len_out", "mass_out", "kept"}}
MAY = {"decode": {("q", "out")}, "prompt": {("q", "out")}, "mass": set(), "evict": {("kv_len", "kv_len_out"), ("mass", "mass_out")}}


def places():
    return {n: STEP * (i + 1) for i, n in enumerate(NAMES)}


def refused(op, **at):
    """The call's status is the refusal; the library's message says why."""
    args = dict(PAGED, ws_bytes=STEP, mass_stride=128, **at)
    return call(op, **args) == _lib.ERR_INVALID_ARG and b"overlap" in _lib.lib().dflash_last_error_string()


@pytest.mark.parametrize("op", ["decode", "prompt", "mass", "evict"])
def test_overlapping_outputs_are_refused(op):
    for a, b in itertools.combinations(USED[op], 2):
        if not {a, b} & WRITTEN[op]:
            continue
        for off in (16, -16) if (a, b) in MAY[op] else (0, 16, -16):
            at = places()
            at[b] = at[a] + off
            assert refused(op, **at), (a, b, off)


def test_evict_refuses_masses_that_share_rows():
    at = places()
    for off in (4, 99, 128 - 99, 127, 128 * 3 + 1):          # rows of 100 floats every 128
        for sign in (1, -1):
            assert refused("evict", **dict(at, mass_out=at["mass"] + 4 * off * sign)), off
