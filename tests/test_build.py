"""The native build reuses what was compiled by the same command from the same sources, and nothing else."""
import os
import stat

import pytest

from tools import build_native as bn


@pytest.fixture
def fake(tmp_path, monkeypatch):
    """A compiler that writes its arguments into its output and counts its calls; one source file."""
    log = tmp_path / "calls"
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\necho "$@" >> %s\nwhile [ $# -gt 0 ]; do\n'
                  '  if [ "$1" = -o ]; then echo made > "$2"; fi\n  shift\ndone\n' % log)
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    src = tmp_path / "csrc" / "kernels"
    src.mkdir(parents=True)
    (src / "a.hip").write_text("// nothing")
    (src / "b.hip").write_text("// nothing")
    (src / "c.h").write_text("// nothing")
    for k, v in (("HIPCC", str(cc)), ("CSRC", str(tmp_path / "csrc")), ("BUILD", str(tmp_path / "build")),
                 ("PKG", str(tmp_path)), ("SOURCES", ["kernels/a.hip", "kernels/b.hip"]), ("HOST_MODULES", [])):
        monkeypatch.setattr(bn, k, v)
    monkeypatch.setattr(bn, "build_h5", lambda verbose=True: None)

    def run():
        """What one build ran: "c" for each compilation, "l" for a link."""
        log.write_text("")
        bn.build(jobs=1, verbose=False)
        return "".join(sorted("c" if " -c " in line else "l" for line in log.read_text().splitlines()))

    return run, tmp_path


def test_unchanged_is_reused(fake):
    run, root = fake
    assert run() == "ccl"
    assert run() == ""
    os.utime(root / "csrc" / "kernels" / "a.hip", (2e9, 2e9))  # newer than its object
    assert run() == "cl"
    os.utime(root / "csrc" / "kernels" / "c.h", (3e9, 3e9))
    assert run() == "ccl"


def test_other_flags_compile_again(fake, monkeypatch):
    run, _ = fake
    run()
    monkeypatch.setattr(bn, "ARCH", "gfx950:sramecc+")
    assert run() == "ccl"
    assert run() == ""


def test_objects_without_a_record_compile_again(fake):
    """An object of a build that kept no record of its command may come from any flags."""
    run, root = fake
    run()
    for name in os.listdir(root / "build"):
        if not name.endswith(".o"):
            os.remove(root / "build" / name)
    assert run() == "ccl"


def test_a_source_less_links_again(fake, monkeypatch):
    run, _ = fake
    run()
    monkeypatch.setattr(bn, "SOURCES", ["kernels/b.hip"])
    assert run() == "l"
    assert run() == ""


def test_a_failed_compilation_leaves_no_record(fake, monkeypatch):
    run, root = fake
    run()
    good = bn.HIPCC
    monkeypatch.setattr(bn, "ARCH", "other")
    monkeypatch.setattr(bn, "HIPCC", "/bin/false")
    with pytest.raises(RuntimeError, match="failed"):
        run()
    monkeypatch.setattr(bn, "HIPCC", good)
    assert run() == "ccl"
