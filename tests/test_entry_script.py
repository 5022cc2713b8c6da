"""The build and smoke script run as a script: what its main block calls stands before it."""
import ast
from pathlib import Path

SCRIPT = Path(__file__).resolve().parent.parent / "__graft_entry__.py"


def _is_main(node):
    return isinstance(node, ast.If) and ast.unparse(node.test) == "__name__ == '__main__'"


def test_the_main_block_is_the_last_statement():
    body = ast.parse(SCRIPT.read_text()).body
    assert [i for i, n in enumerate(body) if _is_main(n)] == [len(body) - 1]


def test_everything_that_the_script_calls_is_defined_when_main_runs():
    """Run as a script with the argument, up to the main block: each module-level name that a function uses is there."""
    tree = ast.parse(SCRIPT.read_text())
    main = next(i for i, n in enumerate(tree.body) if _is_main(n))
    space = {"__name__": "entry", "__file__": str(SCRIPT)}
    exec(compile(ast.Module(tree.body[:main], []), str(SCRIPT), "exec"), space)
    everywhere = {n.name for n in tree.body if isinstance(n, ast.FunctionDef)}
    used = {n.id for n in ast.walk(tree) if isinstance(n, ast.Name) and isinstance(n.ctx, ast.Load)} & everywhere
    assert {"build", "smoke"} <= used and used <= set(space)
