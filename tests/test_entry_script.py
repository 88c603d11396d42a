"""The entry file as a script: whatever its last lines call has been defined above them."""
import ast
import pathlib


def test_nothing_is_defined_behind_the_scripts_own_lines():
    body = ast.parse((pathlib.Path(__file__).parent.parent / "__graft_entry__.py").read_text()).body
    at = [i for i, s in enumerate(body) if isinstance(s, ast.If) and "__main__" in ast.unparse(s.test)]
    assert at == [len(body) - 1], [ast.unparse(s).splitlines()[0] for s in body[at[0] + 1:]]
