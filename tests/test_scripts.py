"""Files that are run as scripts: what follows the block that runs them is not there yet when it runs."""
from __future__ import annotations

import ast
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _is_main(node) -> bool:
    return isinstance(node, ast.If) and ast.unparse(node.test).replace('"', "'") == "__name__ == '__main__'"


def _scripts():
    for path in sorted([*ROOT.glob("*.py"), *(ROOT / "bin").iterdir(), *ROOT.glob("quanta_b200/**/*.py"), *ROOT.glob("parity/*.py")]):
        if path.is_file() and (path.suffix == ".py" or path.read_bytes()[:2] == b"#!" and b"python" in path.read_bytes()[:64]):
            if any(_is_main(n) for n in ast.parse(path.read_text()).body):
                yield pytest.param(path, id=str(path.relative_to(ROOT)))


@pytest.mark.parametrize("path", list(_scripts()))
def test_the_block_that_runs_a_script_is_its_last(path):
    body = ast.parse(path.read_text()).body
    assert _is_main(body[-1]) and sum(map(_is_main, body)) == 1


def test_the_scripts_are_found():
    names = {p.id for p in _scripts()}
    assert {"__graft_entry__.py", "bench.py", "bench_kernels.py"} <= names
