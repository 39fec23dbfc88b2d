"""Order of cluster operations in the kernels' sources, checked on the CPU.

- ``barrier.cluster.*.aligned`` has to be executed by a whole, converged warp. Code behind a
  branch on the thread or lane is not converged by itself, so every function that holds such
  an instruction converges the warp first.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "hopper-lab_b200" / "csrc"


def code(path):
    """A source file without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def body(text, start):
    """The braced block that follows position `start`."""
    i = text.index("{", start)
    depth = 0
    for j in range(i, len(text)):
        depth += {"{": 1, "}": -1}.get(text[j], 0)
        if depth == 0:
            return text[i:j + 1]
    raise AssertionError("unbalanced braces")


def sources():
    return sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def test_warps_converge_before_aligned_cluster_barriers():
    found = 0
    for path in sources():
        text = code(path)
        for m in re.finditer(r"\bvoid (\w+)\([^)]*\) ", text):
            block = body(text, m.end() - 1) if text[m.end()] == "{" else ""
            at = [b.start() for b in re.finditer(r"barrier\.cluster\.\w+[\w.]*\.aligned", block)]
            if at:
                found += 1
                assert "__syncwarp()" in block[:at[0]], f"{path.name}: {m.group(1)}"
        # nowhere outside a small function of its own
        assert len(re.findall(r"barrier\.cluster\.\w+[\w.]*\.aligned", text)) == sum(
            len(re.findall(r"barrier\.cluster\.\w+[\w.]*\.aligned", body(text, m.end() - 1)))
            for m in re.finditer(r"__forceinline__ void \w+\([^)]*\) (?=\{)", text))
    assert found


REMOTE = r"\b(?:mapa_shared|st_shared_cluster\w*|ld_shared_cluster\w*|mbar_arrive_cluster\w*)\s*\("
STARTED = r"\b(?:cluster_sync|cluster_wait)\s*\(\s*\)"


def test_cluster_has_started_before_remote_shared_memory():
    found = 0
    for path in sources():
        text = code(path)
        for m in re.finditer(r"__global__ ", text):
            name = re.search(r"(\w+)\s*\(\s*const", text[m.end():]).group(1)
            block = body(text, m.end())
            remote = re.search(REMOTE, block)
            if remote:
                found += 1
                assert re.search(STARTED, block[:remote.start()]), f"{path.name}: {name}"
    assert found >= 3


def test_block_scaled_products_drain_behind_every_role():
    text = code(CSRC / "mx_gemm.cuh")
    for name, joined in (("mx_gemm_rows_kernel", "__syncthreads()"), ("mx_gemm_pair_kernel", "cluster_sync()")):
        block = body(text, re.search(r"__global__[^{]*\b%s\(" % name, text).end())
        roles_end = block.index(joined, block.index("tmem_wait_ld"))
        drains = [m.start() for m in re.finditer(r"\(i / S\) & 1u", block)]
        assert drains and min(drains) > roles_end, name
