"""The calls of the language model that INTEGRATION.md shows fit the methods' signatures."""

from __future__ import annotations

import ast
import inspect
import re
from pathlib import Path

from double_attention_b200 import DoubleAttentionLM

TEXT = (Path(__file__).parent.parent / "INTEGRATION.md").read_text()


def test_calls_of_the_language_model_bind() -> None:
    seen = set()
    for block in re.findall(r"```python\n(.*?)```", TEXT, re.S):
        for node in ast.walk(ast.parse(block)):
            if not isinstance(node, ast.Call) or not isinstance(node.func, ast.Attribute) or not isinstance(node.func.value, ast.Name):
                continue
            method = vars(DoubleAttentionLM).get(node.func.attr)
            if node.func.value.id != "lm" or method is None:
                continue
            seen.add(node.func.attr)
            inspect.signature(method).bind(None, *node.args, **{k.arg: k.value for k in node.keywords})
    assert {"new_cache", "extend", "score"} <= seen
