"""What the build makes again, and what it leaves: commands are recorded instead of run."""
import os

import pytest

from sequoia_amd import build as B


@pytest.fixture
def made(tmp_path, monkeypatch):
    """-> the list of files that the commands since its last clear() would have written."""
    out = []

    def run(cmd):
        target = cmd[cmd.index("-o") + 1]
        out.append(os.path.basename(target))
        with open(target, "w") as f:
            f.write(" ".join(cmd))

    monkeypatch.setattr(B, "LIBDIR", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libsequoia_hip.so"))
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "_paged.so"))
    monkeypatch.setattr(B, "hipcc", lambda: "hipcc")
    monkeypatch.setattr(B.subprocess, "check_call", run)
    return out


OBJECTS = [s.replace(".hip", ".o") for s in B.SOURCES]


def test_everything_is_made_once(made):
    B.build(verbose=False)
    assert sorted(made) == sorted(OBJECTS + ["libsequoia_hip.so", "_paged.so"])
    made.clear()
    B.build(verbose=False)
    assert made == []
    B.build(force=True, verbose=False)
    assert sorted(made) == sorted(OBJECTS + ["libsequoia_hip.so", "_paged.so"])


def test_other_flags_make_everything_again_that_they_reach(made, monkeypatch):
    B.build(verbose=False)
    made.clear()
    monkeypatch.setattr(B, "FLAGS", B.FLAGS + ["-DANYTHING"])
    B.build(verbose=False)
    assert sorted(made) == sorted(OBJECTS + ["libsequoia_hip.so"])
    made.clear()
    monkeypatch.setattr(B, "EXTRA_FLAGS", {**B.EXTRA_FLAGS, "verify.hip": ["-DMORE"]})
    B.build(verbose=False)
    assert sorted(made) == ["libsequoia_hip.so", "verify.o"]
    made.clear()
    monkeypatch.setattr(B, "SOURCES", B.SOURCES[:-1])
    B.build(verbose=False)
    assert made == ["libsequoia_hip.so"]
    made.clear()
    monkeypatch.setattr(B, "BINDING_FLAGS", B.BINDING_FLAGS + ["-g"])
    B.build(verbose=False)
    assert made == ["_paged.so"]


def test_objects_that_nothing_is_known_of_are_made_again(made, tmp_path):
    B.build(verbose=False)
    made.clear()
    (tmp_path / B.MADE_WITH).unlink()
    B.build(verbose=False)
    assert sorted(made) == sorted(OBJECTS + ["libsequoia_hip.so", "_paged.so"])


def test_a_build_that_ends_early_goes_on_where_it_stopped(made, monkeypatch):
    done = B.subprocess.check_call

    def fails(cmd):
        if any(c.endswith("verify.hip") for c in cmd):
            raise B.subprocess.CalledProcessError(1, cmd)
        done(cmd)

    monkeypatch.setattr(B.subprocess, "check_call", fails)
    with pytest.raises(B.subprocess.CalledProcessError):
        B.build(verbose=False)
    before = list(made)
    assert "verify.o" not in before and "libsequoia_hip.so" not in before
    made.clear()
    monkeypatch.setattr(B.subprocess, "check_call", done)
    B.build(verbose=False)
    assert sorted(before + made) == sorted(OBJECTS + ["libsequoia_hip.so", "_paged.so"])


def test_the_entry_compiles_each_time(made, monkeypatch):
    import __graft_entry__ as entry
    from sequoia_amd import native
    monkeypatch.setattr(native, "load", lambda: None)
    monkeypatch.setattr(native, "load_paged", lambda lib: None)
    for _ in range(2):
        made.clear()
        entry.build()
        assert sorted(made) == sorted(OBJECTS + ["libsequoia_hip.so", "_paged.so"])


def test_without_a_host_compiler_the_library_is_built_all_the_same(made, monkeypatch, tmp_path, capsys):
    from sequoia_amd import native
    B.build(verbose=False)
    run = B.subprocess.check_call

    def fails(cmd):
        if cmd[0] == "no-such-compiler":
            raise FileNotFoundError(cmd[0])
        run(cmd)

    monkeypatch.setenv("CXX", "no-such-compiler")
    monkeypatch.setattr(B.subprocess, "check_call", fails)
    made.clear()
    assert B.build(force=True, verbose=False) == B.LIB
    assert "libsequoia_hip.so" in made and not os.path.exists(B.BINDING) and "_paged.so was not built" in capsys.readouterr().err
    monkeypatch.setattr(native, "PAGED_PATH", B.BINDING)
    with pytest.raises(native.SequoiaNativeError, match="not found"):
        native.load_paged(None)
    monkeypatch.setenv("CXX", "g++")
    made.clear()
    B.build(verbose=False)
    assert made == ["_paged.so"]
