"""The parents of a tree in the Rust binding (source only: no cargo here): an index never reaches the library as
the root's value, HS_TREE_ROOT = u32::MAX."""

import os
import re

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hardshell-hip", "src", "lib.rs")


def test_an_index_is_never_the_root():
    body = re.search(r"fn parents_of\(.*?\n}\n", open(LIB).read(), flags=re.S).group(0)
    assert "unwrap_or(HS_TREE_ROOT))" not in body  # Some(u32::MAX) would pass as the root
    assert "u32::try_from(n).unwrap_or(HS_TREE_ROOT - 1)" in body and "p.map_or(HS_TREE_ROOT, |i| i.min(none))" in body
