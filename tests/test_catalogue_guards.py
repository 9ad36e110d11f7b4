"""What the catalogue operators' sources must say, because no run shows its absence."""

import os

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "movierecommender-tf-trt_amd", "csrc",
                   "ncf_fp8.hip")


def _body(text, head):
    at = text.index(head)
    return text[at:text.index("\n}\n", at)]


def test_staged_tiles_are_waited_for():
    """k_mm_tile's waves read what other waves load straight into LDS: each of its barriers has a wait for the
    wave's own loads ahead of it, written in the source (that a compiler happens to put one there is no promise)."""
    text = open(SRC).read()
    wait = _body(text, "void staged_barrier()")
    assert 0 < wait.index("s_waitcnt vmcnt(0)") < wait.index("__syncthreads()")
    assert '"memory"' in wait
    tile = _body(text, "void k_mm_tile(")
    assert "__syncthreads" not in tile and "s_barrier" not in tile
    assert tile.count("staged_barrier()") == 2
    # and nothing else loads that way
    assert text.count("global_load_lds(") == _body(text, "void stage_rows(").count("global_load_lds(") == 1
    assert text.replace(tile, "").count("stage_rows(") == 1      # (its definition)
