"""What the attention planner chooses for a call, from the built planner itself
(tests/cxx/attention_plan.cpp), so that a test can say which kernels it runs."""
import collections
import os
import subprocess

import _attention as A

EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cxx", "attention_plan")
TYPE = {A.F32: 0, A.F16: 1, A.BF16: 2}
Plan = collections.namedtuple("Plan", "rows target alike slots lists images items tiles grid")


def plan(tokens, heads, kv_heads, dim, count, page=0, columns=0, t=A.F32):
    assert os.path.exists(EXE), "tests/cxx/attention_plan missing: run __graft_entry__.build()"
    r = subprocess.run([EXE, *map(str, (tokens, heads, kv_heads, dim, count, page, columns, TYPE[t]))], capture_output=True,
                       text=True, timeout=60, check=True)
    return Plan(*map(int, r.stdout.split()))


def plan_of(batch, heads, kv_heads, dim, t):
    """The plan of a call over a cache"""
    return plan(batch.tokens, heads, kv_heads, dim, len(batch.new), batch.page, batch.columns, t)
