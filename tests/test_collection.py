"""Every test is collected: a second definition of a name hides the first one without
a word, in a module or in a class."""

import ast
import collections
import os

import pytest

TESTS = os.path.dirname(os.path.abspath(__file__))
MODULES = sorted(f for f in os.listdir(TESTS) if f.endswith(".py"))

# name defined twice -> the module and name under which what is hidden is run
RUN_ELSEWHERE = {
    ("test_gpu_rms_norm.py", "test_many_rows"):
        ("test_gpu_rms_norm_rows.py", "test_rows_on_both_sides_of_the_workgroups"),
}


def _parsed(module):
    with open(os.path.join(TESTS, module), encoding="utf-8") as f:
        return ast.parse(f.read())


def _names(body):
    return collections.Counter(n.name for n in body if isinstance(
        n, (ast.FunctionDef, ast.AsyncFunctionDef, ast.ClassDef)))


def _twice(tree):
    """Names that a module, or a class in it, defines more than once."""
    bodies = [tree.body] + [n.body for n in ast.walk(tree) if isinstance(n, ast.ClassDef)]
    return [name for body in bodies for name, n in _names(body).items() if n > 1]


@pytest.mark.parametrize("module", MODULES)
def test_no_name_is_defined_twice(module):
    for name in _twice(_parsed(module)):
        assert (module, name) in RUN_ELSEWHERE, f"{module} defines {name} twice: the first never runs"


def test_what_is_hidden_runs_elsewhere():
    for (module, name), (other, stands_in) in RUN_ELSEWHERE.items():
        hidden = next(n for n in _parsed(module).body if getattr(n, "name", None) == name)
        run, = [n for n in _parsed(other).body if getattr(n, "name", None) == stands_in]
        same = [[ast.dump(d) for d in n.decorator_list + n.body] for n in (hidden, run)]
        assert same[0] == same[1]


def test_a_second_definition_is_seen():
    assert _twice(ast.parse("def a(): pass\ndef b(): pass\n")) == []
    assert _twice(ast.parse("def a(): pass\ndef a(x): pass\n")) == ["a"]
    assert _twice(ast.parse("class A:\n  def t(self): pass\n  def t(self): pass\n")) == ["t"]
