"""Guards on the sources and the compiler's output of kernels that address LDS copies through m0 and count their
outstanding vector memory operations."""
import re

import pytest

from sparse_amd import build


def test_inline_assembly_that_writes_m0_says_so():
    """The compiler keeps what it put into m0 unless a statement that writes it lists it as overwritten."""
    seen = 0
    for path in sorted(build.CSRC.glob("*.hip")) + sorted(build.CSRC.glob("*.h")):
        for statement in re.findall(r"asm\s+volatile\s*\((.*?)\)\s*;", path.read_text(), flags=re.S):
            if re.search(r"s_mov_b32 m0\b", statement):
                seen += 1
                assert '"m0"' in statement.rsplit(":", 1)[-1], (path.name, statement)
    assert seen >= 3


# per source: kernel, {(tile height / 32, narrow): slabs requested ahead}, copies a slab for each 32 rows, matrix
# instructions for each 16 x 16 tile and slab, instantiations
COUNTED = {"fp8_tile.hip": ("f8_tile_kernel", {(1, True): 6, (1, False): 4, (2, False): 3, (3, False): 2, (4, False): 2}, 1, 1, 4),
           "fp8_gateup.hip": ("f8_gateup_kernel", {(1, False): 4, (2, False): 3, (3, False): 1, (4, False): 1}, 2, 4, 1)}


@pytest.mark.parametrize("source", list(COUNTED))
def test_tiles_issue_their_vector_memory_operations_as_the_counted_waits_assume(tmp_path, source):
    """Before the barrier that closes a k slab the 8-bit tile kernels wait for all but the newest vector memory
    operations: those of its own fragments and of the slabs requested since.  That is exact only if every slab issues, in
    this order, its LDS copies and two fragment loads for each group of 16 weight rows, and nothing else that the counter
    counts, or, behind the loop, nothing at all.  Checked on the compiler's output for every height, format and kind of
    scales; a slab's height is told by its matrix instructions."""
    import subprocess
    kernel, depth, copies, instructions, forms = COUNTED[source]
    out = tmp_path / "kernel.s"
    cmd = [build._hipcc(), *[f for f in build.HIP_FLAGS if f != "-fPIC"], f"-I{build.INCLUDE}", f"-I{build.CSRC}", "-S",
           "--cuda-device-only", str(build.CSRC / source), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-2000:]
    found, name, segment = {}, None, []
    for line in out.read_text().splitlines():
        m = re.match(r"^(_Z\w+):", line)
        if m:
            name, segment = m.group(1), []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif re.match(r"^\.LBB\d+_\d+:", line):
            segment = []
        text = line.strip().split(";")[0].strip()
        if name is None or kernel not in name or not text or text.startswith(".") or text.endswith(":"):
            continue
        if not text.startswith("s_barrier"):
            segment.append(text)
            continue
        products = sum(i.startswith("v_mfma") for i in segment)
        if products:
            narrow = "ELb1EEEv" in name
            groups = 2 if narrow else 4
            height, rest = divmod(products, 2 * groups * instructions)
            assert rest == 0 and (height, narrow) in depth, (name, products)
            vm = [i for i in segment if i.startswith(("global_", "scratch_", "buffer_", "flat_"))]
            kinds = ["copy" if i.startswith("global_load_lds_dwordx4") else
                     "fragment" if i.startswith("global_load_dwordx4") else i for i in vm]
            waits = [(k, int(re.search(r"vmcnt\((\d+)\)", i).group(1))) for k, i in enumerate(segment)
                     if i.startswith("s_waitcnt") and "vmcnt" in i]
            assert waits and waits[-1][0] > max(k for k, i in enumerate(segment) if i in vm or i.startswith("v_mfma"))
            if kinds:
                assert kinds == ["copy"] * (copies * height) + ["fragment"] * (2 * groups), (name, height, kinds)
            found.setdefault(name, {}).setdefault(height, []).append((bool(kinds), waits[-1][1]))
        segment = []
    assert len(found) == forms
    for name, heights in found.items():
        narrow = "ELb1EEEv" in name
        assert set(heights) == {h for h, n in depth if n == narrow}, (name, set(heights))
        for h, slabs in heights.items():
            S, loads = depth[h, narrow], 4 if narrow else 8
            # the next slab's fragments, then copies and fragments of the slabs requested behind it: S - 1 in the loop,
            # S - 2 - j in number j behind it; each once for scales that are powers of two and once for others
            want = [(True, loads + (S - 1) * (copies * h + loads))] * S
            want += [(False, loads + (S - 2 - j) * (copies * h + loads)) for j in range(S - 1)]
            assert sorted(slabs) == sorted(2 * want), (name, h, slabs)
