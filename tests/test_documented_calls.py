"""The calls of this package that the documents' examples make: each takes the arguments that it is given there."""
from __future__ import annotations

import ast
import importlib
import inspect
import re
import textwrap
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PACKAGE = "latent_bounded_interfaces_amd"


def _examples():
    for path in sorted(ROOT.glob("*.md")):
        for i, block in enumerate(re.findall(r"^```python\n(.*?)^```", path.read_text(), re.S | re.M)):
            if PACKAGE in block:
                yield pytest.param(textwrap.dedent(block), id=f"{path.stem}-{i}")


def _calls(source):
    """(function of the package, call) for each call of an imported name."""
    tree = ast.parse(source)
    known = {}
    for node in ast.walk(tree):
        if isinstance(node, ast.ImportFrom) and (node.module or "").startswith(PACKAGE):
            module = importlib.import_module(node.module)
            known.update({name.asname or name.name: getattr(module, name.name) for name in node.names})
    for node in ast.walk(tree):
        if isinstance(node, ast.Call) and isinstance(node.func, ast.Name) and node.func.id in known:
            yield known[node.func.id], node


@pytest.mark.parametrize("source", _examples())
def test_arguments_of_examples(source):
    for function, call in _calls(source):
        if any(isinstance(a, ast.Starred) for a in call.args) or any(k.arg is None for k in call.keywords):
            continue
        inspect.signature(function).bind(*call.args, **{k.arg: k.value for k in call.keywords})


def test_there_are_examples():
    assert sum(1 for example in _examples() for _ in _calls(example.values[0])) >= 4
