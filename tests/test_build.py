"""What a build leaves behind, with a compiler that only writes files."""

import os
import stat

import pytest

from fsctep_amd import build as B

FAKE = """#!/bin/sh
for a in "$@"; do
  case "$a" in */{fails}) bad=1;; esac
  if [ "$last" = -o ]; then out="$a"; fi
  last="$a"
done
echo made > "$out"
[ -z "$bad" ]
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Compilers, and the places that a build writes to, in a folder of their own; the libraries of a build before."""
    for name in ("pkg", "cpp", "bin"):
        (tmp_path / name).mkdir()
    places = dict(PKG=tmp_path / "pkg", LIB=tmp_path / "pkg" / "libfsctep_hip.so", TORCH_LIB=tmp_path / "pkg" / "libfsctep_torch.so",
                  CORE_RUN=tmp_path / "cpp" / "core_run")
    for name, place in places.items():
        monkeypatch.setattr(B, name, str(place))
        if name != "PKG":
            place.write_text("before")

    def fails(source):
        for name in ("hipcc", "g++"):
            script = tmp_path / "bin" / name
            script.write_text(FAKE.format(fails=source))
            script.chmod(script.stat().st_mode | stat.S_IXUSR)
        monkeypatch.setenv("HIPCC", str(tmp_path / "bin" / "hipcc"))
        monkeypatch.setenv("PATH", f"{tmp_path / 'bin'}{os.pathsep}{os.environ['PATH']}")
        return places

    return fails


def files():
    return sorted(os.path.join(d, f) for top in (B.PKG, B.CSRC, os.path.dirname(B.CORE_RUN)) for d, _, fs in os.walk(top) for f in fs)


# a HIP source, a torch source, the program, either library's link
@pytest.mark.parametrize("source", ["layer_norm.hip", "torch_ops.cpp", "core_run.cpp", "adamw.hip.o", "torch_learn_ops.o"])
def test_a_build_that_fails_leaves_nothing(tree, source):
    places, before = tree(source), files()
    with pytest.raises(RuntimeError, match="failed"):
        B.build()
    assert files() == before and os.listdir(B.CSRC)
    assert all(places[k].read_text() == "before" for k in ("LIB", "TORCH_LIB", "CORE_RUN"))


def test_a_build_leaves_the_libraries_alone(tree):
    places, before = tree("nothing"), files()
    assert B.build() == B.LIB and files() == before
    assert all(places[k].read_text() == "made\n" for k in ("LIB", "TORCH_LIB", "CORE_RUN")) and not os.path.exists(os.path.join(B.PKG, "_build"))
