"""CPU checks at the edges of the packed-batch operators: size calls, and the calls that the performance cases make."""

import ast
import inspect
import os

import pytest

import fn

CASES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


@pytest.mark.parametrize("B,T,nkh,nvh", [(1, 64, 2, 4), (3, 700, 16, 48)])
def test_chunk_workspace_of_core_and_block(fnlib, B, T, nkh, nvh):
    """The workspace of the core and of the block, asked for by name or by place."""
    core = fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh)
    assert core > 0
    assert core == fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh, False) == fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh, True)
    assert core == fnlib.gdn_chunk_work_bytes(B, T, nkh, nvh, block=True)


# entries of a call's *_p(...) argument count one each
def _places(call):
    n = 0
    for a in call.args:
        n += len(a.value.args) if isinstance(a, ast.Starred) else 1
    return n


def test_performance_cases_call_what_there_is():
    """Every call of the library in the performance cases fits its method's arguments."""
    seen = set()
    for node in ast.walk(ast.parse(open(CASES).read())):
        if not (isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) and hasattr(fn.FN, node.func.attr)):
            continue
        of = node.func.value
        if not (isinstance(of, ast.Name) and of.id == "L" or isinstance(of, ast.Call) and getattr(of.func, "id", "") == "lib"):
            continue
        inspect.signature(getattr(fn.FN, node.func.attr)).bind(None, *[0] * _places(node), **{k.arg: 0 for k in node.keywords})
        seen.add(node.func.attr)
    assert {"page_plan_dev", "attn_kv4_dev", "gdn_chunk_work_bytes", "gdn_core_chunk_dev", "gdn_block_chunk_dev"} <= seen


@pytest.mark.parametrize("call", ["kv4_pack_dev", "kv4_unpack_dev"])
def test_more_rows_than_a_launch_has_are_refused(fnlib, call):
    with pytest.raises(RuntimeError, match="n must be <= 33554431"):
        getattr(fnlib, call)(1 << 25, 1, 4, 4096, *[4096] * 3)


def test_more_chunks_than_a_launch_has_are_refused(fnlib):
    """Before any work is launched: workgroups of the preparation, and of the block's gated norm."""
    T, p = 1 << 30, 4096
    with pytest.raises(RuntimeError, match="too many rows"):
        fnlib.gdn_core_chunk_dev(1, T, 1, 1, *[p] * 9, 1 << 60)
    T = 1 << 23
    with pytest.raises(RuntimeError, match="too many rows"):
        fnlib.gdn_block_chunk_dev(1, T, 1, 16, 4, *[p] * 13, 1 << 60)
