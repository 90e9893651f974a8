"""Source checks of the bounded waits in the grouped and adapter kernels.  A wait that ran
out cannot be had on a GPU without stopping one, so what it relies on is read:
the lanes of a role agree on the outcome, polling ends, and copies in flight
are awaited once every role of the CTA has stopped."""
from __future__ import annotations

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "veystrix-core_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


def body(text, head):
    """The braces' contents after the first place that `head` matches."""
    at = text.index("{", re.search(head, text).end())
    depth, end = 1, at + 1
    while depth:
        depth += {"{": 1, "}": -1}.get(text[end], 0)
        end += 1
    return text[at + 1:end - 1]


def test_the_lanes_of_a_role_agree_on_a_wait():
    wait = body(source("vx_grouped.cuh"), r"bool role_wait\(")
    last = wait.index("__all_sync(0xFFFFFFFFu")
    # nothing is returned, and nobody is told to stop, before the vote
    assert "return" not in wait[:last] and "*dead = 1" not in wait[:last]
    assert "return" in wait[last:]


@pytest.mark.parametrize("name", ["vx_grouped.cu", "vx_grouped_mid.cu"])
def test_copies_in_flight_are_awaited_after_all_roles(name):
    text = source(name)
    kernel = body(text, r"__launch_bounds__\(k\w+Threads, 1\)\s*\n?\s*grouped\w*_kernel\(")
    roles_end = kernel.rindex("__syncthreads()")
    drain = kernel.index("let the copies in flight land")
    assert drain > roles_end and "kWaitLimitNs" in kernel[drain:]
    assert drain < kernel.index("dealloc", drain), "before the CTA gives up its memory"


@pytest.mark.parametrize("name", sorted(n for n in os.listdir(CSRC) if n.startswith(("vx_grouped", "vx_lora"))))
def test_polling_loops_have_a_limit(name):
    text = source(name)
    for m in re.finditer(r"while \(!mbar_try\((?:[^()]|\([^()]*\))*\)", text):
        assert "kWaitLimitNs" in text[m.start():m.start() + 300]
    for m in re.finditer(r"for \([^;]*; i < kSpinLimit", text):
        assert "kWaitLimitNs" in text[m.start():m.start() + 600]


def test_adapter_parts_on_their_way_are_awaited_before_the_cta_leaves():
    """Peers store into this CTA's shared memory: one that gave up stays for them."""
    text = source("vx_lora.cu")
    kernel = body(text, r"lora_small_kernel\(const LoraArgs a\)")
    assert re.search(r"const bool ok = lora_wait\(&arrived\);\s*if \(!ok\) lora_wait\(&arrived\);", kernel)
