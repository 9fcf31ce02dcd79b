"""Streams of different priorities have hung for good where work on them waited for each other: the package makes none."""
import ast
import os

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def sources(*suffixes):
    for top in ("sequoia_amd", "benchmarks"):
        for where, _, files in os.walk(os.path.join(REPO, top)):
            yield from (os.path.join(where, f) for f in files if f.endswith(suffixes))
    if ".py" in suffixes:
        yield os.path.join(REPO, "bench.py")


def test_no_stream_is_given_a_priority():
    seen = 0
    for path in sources(".py"):
        with open(path) as f:
            for call in ast.walk(ast.parse(f.read())):
                if isinstance(call, ast.Call):
                    seen += 1
                    assert not {"priority", "is_high_priority_stream"} & {k.arg for k in call.keywords}, f"{path}:{call.lineno}"
    assert seen > 1000
    for path in sources(".hip", ".h", ".cpp"):
        with open(path) as f:
            assert "StreamCreateWithPriority" not in f.read(), path
