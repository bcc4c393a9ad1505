"""The documents' usage examples, read as code: every call of this module has arguments that its function takes, and
what comes together stays together."""
import ast
import inspect
import re

import pytest
from conftest import ROOT

import qwen_kernels_gpu as qk

EXAMPLES = [(p.name, m.group(1)) for p in sorted(ROOT.glob("*.md"))
            for m in re.finditer(r"^```python\n(.*?)^```", p.read_text(), re.M | re.S) if "import qwen_kernels_gpu" in m.group(1)
            or "qk." in m.group(1)]


def calls_of(text):
    """(name, call) of the module's functions."""
    for x in ast.walk(ast.parse(text)):
        if isinstance(x, ast.Call) and isinstance(x.func, ast.Attribute) and getattr(x.func.value, "id", "") == "qk":
            yield x.func.attr, x


@pytest.mark.parametrize("name,text", EXAMPLES, ids=[f"{n}-{i}" for i, (n, _) in enumerate(EXAMPLES)])
def test_calls_fit_their_functions(name, text):
    for f, call in calls_of(text):
        inspect.signature(getattr(qk, f)).bind(*call.args, **{k.arg: k.value for k in call.keywords})


@pytest.mark.parametrize("name,text", EXAMPLES, ids=[f"{n}-{i}" for i, (n, _) in enumerate(EXAMPLES)])
def test_frequencies_go_with_their_amplitude(name, text):
    """rotary_frequencies gives both: whatever is rotated by the one is multiplied by the other, or a long context's
    queries and keys do not fit one another."""
    if "freqs, amplitude = " not in text:
        return
    turned = 0
    for f, call in calls_of(text):
        given = inspect.signature(getattr(qk, f)).bind(*call.args, **{k.arg: k.value for k in call.keywords}).arguments
        if getattr(given.get("freqs"), "id", "") == "freqs":
            turned += 1
            assert getattr(given.get("amplitude"), "id", "") == "amplitude", ast.unparse(call)
    assert turned


def test_there_are_examples():
    assert any("kv_cache_append" in text for _, text in EXAMPLES)
