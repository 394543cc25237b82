"""The attention kernels' warp-wide instructions (`.aligned`: tcgen05.ld/st and
their waits, ldmatrix, mma.sync, bar.sync, the cluster's barrier, setmaxnreg)
want a warp whose lanes run together. Behind a branch that lanes take
differently, a lane's own wait included, the source therefore has an explicit
warp or block barrier before the next of them. Read off the source, every loop
walked twice so that its end is followed by its start; what stands before a
`break` does not lead on."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parents[1] / "ggml-xdna_b200" / "csrc" / "attend.cu"

ALIGNED = re.compile(r"\b(tmem_(ld|st)\w*|tmem_(alloc|dealloc|relinquish)|ldmatrix_x4(_t)?|mma16816(<\w+>)?|named_barrier"
                     r"|cluster_sync)\(|setmaxnreg")
TOGETHER = re.compile(r"\b(__syncwarp|__syncthreads|warp_arrive)\(")
LANES = (r"lane|threadIdx\.x|elect_one\(\)|tq == 0|mine|has|valid|found|bad|bad_half<F16>|any_bad<F16>|row|rows|live|key|seen|e")  # what differs from lane to lane
PARTS = re.compile(rf"\b(if|while) \(.*(?<!\w)({LANES})(?!\w)|\bfor \(.*(threadIdx\.x|= row;|= lane)|mbar_wait_bounded\(")


def lines_of(kernel: str) -> list[tuple[int, str]]:
    """The kernel's lines without comments, by number."""
    text = SOURCE.read_text().split("\n")
    start = next(i for i, s in enumerate(text) if re.search(rf"\b{kernel}\(", s))
    end = next(i for i in range(start, len(text)) if text[i] == "}")
    return [(i + 1, re.sub(r"//.*", "", text[i])) for i in range(start, end)]


def block_end(lines: list[tuple[int, str]], i: int) -> int:
    indent = len(lines[i][1]) - len(lines[i][1].lstrip())
    return next(k for k in range(i + 1, len(lines)) if lines[k][1].startswith(" " * indent + "}"))


def walked(lines: list[tuple[int, str]]) -> list[tuple[int, str]]:
    """In the order they run, a loop's body twice."""
    out, i = [], 0
    while i < len(lines):
        n, s = lines[i]
        if re.match(r"\s*(for|while) \(.*\{\s*$", s):
            j = block_end(lines, i)
            body = walked(lines[i + 1:j])
            out += [(n, s)] + body + body
            i = j
        elif re.match(r"\s*if \(.*\{\s*$", s) and lines[(j := block_end(lines, i)) - 1][1].strip() == "break;":
            out.append((n, s))
            i = j + 1
        else:
            out.append((n, s))
            i += 1
    return out


def unjoined(kernel: str) -> list[str]:
    """Warp-wide instructions that a lane's branch may lead to without a barrier between."""
    parted, found = None, {}
    for n, s in walked(lines_of(kernel)):
        # what a line does, left to right
        marks = [(m.start(), kind) for kind, rx in (("parts", PARTS), ("together", TOGETHER), ("aligned", ALIGNED))
                 for m in rx.finditer(s)]
        for _, kind in sorted(marks):
            if kind == "parts":
                parted = n
            elif kind == "together":
                parted = None
            elif parted is not None:
                found[n] = f"line {n}: {s.strip()} (lanes part on line {parted})"
    return list(found.values())


def test_few_rows():
    assert unjoined("kv_attend_few_kernel") == []


def test_many_rows():
    assert unjoined("kv_attend_many_kernel") == []


def test_waits_leave_a_warp_together():
    for name in ("wait_on", "warp_arrive"):
        body = [s for _, s in lines_of(name)]
        last = max(i for i, s in enumerate(body) if "__syncwarp()" in s)
        assert not any(PARTS.search(s) for s in body[last + 1:] if "__all_sync" not in s)
