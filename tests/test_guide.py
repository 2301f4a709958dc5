"""INTEGRATION.md against the package: what it calls is there, and its markup is whole."""
from __future__ import annotations

import inspect
import re

import pytest

from conftest import REPO_ROOT, import_submodule

GUIDE = (REPO_ROOT / "INTEGRATION.md").read_text()
FENCE = re.compile(r"^```(\w*)\n(.*?)^```$", re.S | re.M)
BLOCKS = [code for lang, code in FENCE.findall(GUIDE) if lang == "python"]
PROSE = [line for line in FENCE.sub("", GUIDE).splitlines() if line.strip()]


def test_code_spans_are_closed():
    assert [line for line in PROSE if line.count("`") % 2] == []


@pytest.mark.parametrize("code", BLOCKS, ids=range(len(BLOCKS)))
def test_blocks_are_python_and_their_operators_exist(code):
    compile(code, "INTEGRATION.md", "exec")
    ops = import_submodule("ops")
    assert [name for name in re.findall(r"\bops\.(\w+)", code) if not hasattr(ops, name)] == []


def test_operators_with_a_workspace_are_named():
    """The sentence on workspaces names each operator over the 8-bit layer that takes one, and what sizes it."""
    ops = import_submodule("ops")
    spans = {s for line in PROSE if "`workspace=`" in line and "gqa_kv8" in line for s in re.findall(r"`([^`]+)`", line)}
    takes = [n for n, f in vars(ops).items() if inspect.isfunction(f) and not n.startswith("_")
             and "workspace" in inspect.signature(f).parameters and n.startswith(("linear_int8", "gqa_kv8", "token_"))]
    assert len(takes) == 5
    assert [n for n in takes if n not in spans or f"{n}_workspace_bytes" not in spans] == []


def test_trees_and_windows_are_apart():
    """The windowed form's mask goes by places: rows of a drafted tree would see drafts that are not their ancestors."""
    drafted = [code for code in BLOCKS if "ops.gqa_kv8_tree(" in code]
    assert drafted and not any("ops.gqa_kv8_window(" in code for code in drafted)
    assert any("ops.gqa_kv8_window(" in code for code in BLOCKS)
    assert "tree" in import_submodule("ops").gqa_kv8_window.__doc__
