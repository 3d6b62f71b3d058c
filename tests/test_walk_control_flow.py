"""The loops of verify's walk, in the instructions that the compiler makes of it (no GPU needed)."""
import re
import subprocess

from tinygiant_amd import build as B


def test_no_loop_of_the_walk_is_left_lane_by_lane(tmp_path):
    """A loop that lanes leave one after the other takes them out of exec until none is left (s_andn2_b64 exec, exec).
    Behind such loops the compiler placed register copies where all lanes are off; the walk and what it is called by
    have none, so that no such copy can be lost."""
    out = tmp_path / "draft.s"
    subprocess.run([B.HIPCC, *B.HIP_FLAGS, *B.EXTRA_FLAGS["tg_draft.hip"], "--cuda-device-only", "-S", str(B.CSRC / "tg_draft.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    kernel, loops = None, {}
    for line in out.read_text().splitlines():
        name = re.match(r"(_ZN2tg\w+):", line)
        if name:
            kernel = name[1]
            loops[kernel] = 0
        elif kernel and re.search(r"\bs_andn2_b64 exec, exec\b", line):
            loops[kernel] += 1
    walks = {k: n for k, n in loops.items() if "k_verify_walk" in k or "k_verify_sweep" in k}
    assert len(walks) == 6 and not any(walks.values()), loops
