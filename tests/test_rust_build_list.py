"""The crate's build script, which is not compiled here, against the library's own build."""
import os
import re

from wick_b200 import build

RUST = os.path.join(os.path.dirname(build.__file__), "rust")


def test_the_crate_compiles_the_same_sources():
    text = open(os.path.join(RUST, "build.rs")).read()
    sources = re.findall(r'"([^"]+\.cu)"', re.search(r"const SOURCES: &\[&str\] = &\[(.*?)\];", text, re.S).group(1))
    assert sources == build.SOURCES
    assert all(os.path.exists(os.path.join(build.CSRC, s)) for s in sources)


def test_the_crate_is_built_anew_when_a_header_changes():
    assert re.search(r"rerun-if-changed=\{\}\", src_dir\.display\(\)", open(os.path.join(RUST, "build.rs")).read())
