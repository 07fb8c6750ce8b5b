"""Rules of the attention's copies that no GPU test can break safely: checked in the sources."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "miniworld_b200" / "csrc"


def test_copying_threads_wait_for_their_copies_before_they_leave():
    """Another warp may give up after the copying thread has started its last copy: whether one has by then says nothing about the copies
    in flight, so the wait for them does not hang on it (every such wait is bounded)."""
    found = 0
    for name in ("attention_forward.cuh", "attention_backward.cuh"):
        lines = [line.split("//")[0].rstrip() for line in (CSRC / name).read_text().splitlines()]
        for i, line in enumerate(lines):
            if "state.drain<" in line:
                found += 1
                assert re.fullmatch(r"\s*state\.drain<ST>\(\w+, landed, ready\);", line), line
                assert lines[i - 1].strip() == "}" and lines[i + 1].strip().startswith("} else if (warp == mma_warp"), (lines[i - 1], lines[i + 1])
    assert found == 3
    tiles = (CSRC / "attention_tiles.cuh").read_text()
    drain = tiles[tiles.index("void drain(") :]
    assert "kWaitLimitCycles" in drain[: drain.index("\n  }\n")]
