"""build() on the CPU, its compilers stood in for by small scripts."""
import os
import stat
import sys
import time

import pytest


@pytest.fixture
def built(monkeypatch, tmp_path):
    """(build, its library, its _dispatch.so): both there from an earlier build, in a folder of their own."""
    from shard_amd import build as b
    cc = tmp_path / "hipcc"
    cc.write_text(f"#!{sys.executable}\n"
                  "import os, sys\n"
                  "out = sys.argv[sys.argv.index('-o') + 1]\n"
                  "if os.environ.get('STUB_FAILS') in (('link', 'all') if '-shared' in sys.argv else ('compile', 'all')):\n"
                  "    sys.exit('no')\n"
                  "open(out, 'w').write('new')\n")
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    lib, dispatch = tmp_path / "lib.so", tmp_path / "_dispatch.so"
    lib.write_text("old")
    dispatch.write_text("old")
    monkeypatch.setattr(b, "hipcc", lambda: str(cc))
    monkeypatch.setattr(b, "LIB", str(lib))
    monkeypatch.setattr(b, "DISPATCH", str(dispatch))
    monkeypatch.setattr(b, "dispatch_command", lambda out: [str(cc), "-o", out, "-c"])
    return b, lib, dispatch


def test_both_are_replaced(built):
    b, lib, dispatch = built
    assert b.build() == str(lib)
    assert lib.read_text() == dispatch.read_text() == "new"
    assert sorted(f for f in os.listdir(lib.parent)) == ["_dispatch.so", "hipcc", "lib.so"]


@pytest.mark.parametrize("how", ["fails", "no compiler", "no torch"])
def test_the_library_is_built_without_the_compiled_calls(built, monkeypatch, capfd, how):
    """A warning, and no _dispatch.so of an earlier build beside the new library."""
    b, lib, dispatch = built

    def command(out):
        if how == "no torch":
            raise ImportError("torch")
        return ["/nowhere/g++"] if how == "no compiler" else [sys.executable, "-c", "import sys; print('broken'); sys.exit(1)"]
    monkeypatch.setattr(b, "dispatch_command", command)
    assert b.build() == str(lib)
    assert lib.read_text() == "new" and not dispatch.exists()
    assert "_dispatch.so not built" in capfd.readouterr().err


@pytest.mark.parametrize("fails", ["compile", "link"])
def test_a_failed_build_leaves_what_was_there(built, monkeypatch, tmp_path, fails):
    """Both files as they were, and nothing left running."""
    b, lib, dispatch = built
    pid = tmp_path / "pid"
    monkeypatch.setenv("STUB_FAILS", fails)
    monkeypatch.setattr(b, "dispatch_command", lambda out: [
        sys.executable, "-c", f"import os, time; open({str(pid)!r} + '_', 'w').write(str(os.getpid())); "
                              f"os.rename({str(pid)!r} + '_', {str(pid)!r}); time.sleep(60)"])
    sources = b.sources()

    def after_the_start():  # the compiled calls' compiler runs by then
        for _ in range(2000):
            if pid.exists():
                break
            time.sleep(0.01)
        return sources
    monkeypatch.setattr(b, "sources", after_the_start)
    with pytest.raises(RuntimeError):
        b.build()
    assert lib.read_text() == dispatch.read_text() == "old"
    with pytest.raises(ProcessLookupError):
        os.kill(int(pid.read_text()), 0)
