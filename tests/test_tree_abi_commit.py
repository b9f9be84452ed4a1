"""dsr_commit_tree's argument errors around the caches' addresses and the state
before the step, without a GPU."""
import ctypes

import pytest

from deepseekrpc_amd import _native as N


def arguments():
    a = N.CommitArgs()
    for i, f in enumerate(("parents", "tokens_in", "sampled", "offsets", "kv_lengths", "table", "output_limit", "path",
                           "ids", "accepted", "count", "pending", "stop", "lengths", "status")):
        setattr(a, f, 4096 * (i + 1))
    a.requests, a.tokens, a.table_ld, a.width, a.page, a.blocks = 2, 8, 4, 4, 16, 9
    a.cache_count, a.heads, a.row_bytes, a.c_block, a.c_token, a.c_head = 3, 2, 256, 8192, 512, 256
    return a


@pytest.mark.parametrize("fields", [dict(), dict(caches=4096, host_caches=4096),
                                    dict(caches=4096, lengths_in=4), dict(caches=4096, pending_in=4, plan_status=4),
                                    dict(caches=4096, lengths_in=4, pending_in=4)])
def test_refused(fields):
    a = arguments()
    for f, v in fields.items():
        setattr(a, f, v)
    assert N.load().dsr_commit_tree(ctypes.byref(a), None) == -1


@pytest.mark.parametrize("field,output", [("lengths_in", "lengths"), ("pending_in", "pending"),
                                          ("plan_status", "status")])
def test_the_state_before_the_step_is_no_output(field, output):
    a = arguments()
    a.caches, a.lengths_in, a.pending_in, a.plan_status = 4096, 4, 4, 4
    setattr(a, field, getattr(a, output))
    assert N.load().dsr_commit_tree(ctypes.byref(a), None) == -1


def test_structs_and_the_version_that_gates_them():
    """A library reads whole structs: whoever makes one longer raises the version."""
    sizes = {s: ctypes.sizeof(getattr(N, s)) for s in ("PlanArgs", "RotaryArgs", "TreeAttentionArgs", "CommitArgs")}
    assert (N.ABI_VERSION, sizes) == (7, dict(PlanArgs=184, RotaryArgs=280, TreeAttentionArgs=232, CommitArgs=248))
