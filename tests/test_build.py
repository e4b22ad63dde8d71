"""What the build looks at when it decides whether a library, or a measurement of it, still belongs to the tree."""
import os

from montecarlo_amd import build


def test_measurements_belong_to_the_flags_too(monkeypatch):
    before = build.sources_digest()
    assert before == build.sources_digest()
    for name in ("FLAGS", "LINK_FLAGS"):
        with monkeypatch.context() as m:
            m.setattr(build, name, getattr(build, name)[:-1])
            assert build.sources_digest() != before


def test_a_library_older_than_the_flags_is_built_again(monkeypatch, tmp_path):
    lib = tmp_path / "lib.so"
    monkeypatch.setattr(build, "LIB", str(lib))
    assert build.needs_build()
    lib.write_bytes(b"")
    deps = [os.path.join(build.CSRC, s) for s in build.SOURCES] + build.HEADERS
    newest, flags = max(os.path.getmtime(d) for d in deps), os.path.getmtime(build.__file__)
    os.utime(lib, (max(newest, flags) + 1,) * 2)
    assert not build.needs_build()
    os.utime(lib, (min(newest, flags) - 1,) * 2)
    assert build.needs_build()
    monkeypatch.setattr(build, "SOURCES", [])                # (the flags alone are newer)
    monkeypatch.setattr(build, "HEADERS", [])
    assert build.needs_build()
