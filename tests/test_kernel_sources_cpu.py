"""Rules that the CUDA sources keep and that no run on a healthy GPU can show."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "templar_b200" / "ops" / "csrc"


@pytest.mark.parametrize("src", sorted(p.name for p in CSRC.glob("*.cu")))
def test_drains_do_not_wait_on_the_shared_flag(src):
    """A wait whose result nobody looks at is a drain: it stands in front of a role's return so that no copy lands in shared
    memory that the CTA has given back.  With the CTA's own flag, which is up exactly when a role has given up, ``mbar_wait``
    returns at once, so a drain goes through ``Drain``."""
    text = re.sub(r"//[^\n]*", "", (CSRC / src).read_text())
    # a statement that starts with the call: after a brace, a semicolon or a loop head
    ignored = re.findall(r"(?:[;{}]|\bfor \([^{}]*\))\s*(mbar_wait\([^;]*);", text)
    assert not ignored, ignored


@pytest.mark.parametrize("src", sorted(p.name for p in CSRC.glob("*.cu") if "mbar_expect_tx(" in p.read_text()))
def test_every_kernel_that_asks_for_copies_drains_them(src):
    """Each kernel that arms a barrier for bulk copies waits for them before its CTA retires."""
    text = re.sub(r"//[^\n]*", "", (CSRC / src).read_text())
    kernels = re.split(r"__global__", text)[1:]
    arming = [k for k in kernels if "mbar_expect_tx(" in k.split("<<<")[0]]
    assert arming
    for k in arming:
        assert "Drain drain" in k, k[:200]


def _kernels(src):
    """(name, parameter list, body) of every kernel of a source file."""
    text = re.sub(r"//[^\n]*", "", (CSRC / src).read_text())
    for m in re.finditer(r"__global__[^;{]*?(\w+)\s*\(([^(){}]*)\)\s*\{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield m.group(1), m.group(2), text[m.end():i]


@pytest.mark.parametrize("src", sorted(p.name for p in CSRC.glob("*.cu") if "grid_wait();" in p.read_text()))
def test_restrict_pointers_are_taken_anew_behind_the_grid_wait(src):
    """A kernel that may start while the one before it runs touches no memory before ``grid_wait``.  The compiler may move an
    access through a ``__restrict__`` pointer across the wait unless the pointer goes through ``behind_grid_wait`` there, those
    that are written and read as well as the constant ones."""
    waiting = [k for k in _kernels(src) if "grid_wait();" in k[2]]
    assert waiting
    for name, params, body in waiting:
        pointers = re.findall(r"__restrict__\s+(\w+)", params)
        before, behind = body.split("grid_wait();", 1)
        taken = set(re.findall(r"behind_grid_wait\((\w+)\)", behind))
        assert set(pointers) <= taken, (name, set(pointers) - taken)
        assert not any(re.search(rf"\b{p}\b", before) for p in pointers), name


def test_every_exit_of_a_loss_kernel_has_written_its_row():
    """The mean is taken over the rows' array whatever it holds, and the entry that must not allocate has no status word, so a
    kernel that writes rows of losses has neither a wait that can run out nor a ``return`` in front of the row's loss."""
    kernels = [k for k in _kernels("elementwise.cu") if re.search(r"\blosses\[\w+\] = ", k[2])]
    assert len(kernels) == 2
    for name, _, body in kernels:
        assert "mbar_wait" not in body, name
        for exit_at in re.finditer(r"\breturn;", body):
            assert re.search(r"\blosses\[row\] = ", body[:exit_at.start()]), name


def _agreement_steps(text):
    """What one warp does in ``quadrant_agrees``, in order: "raise" its flag where its wait gave up, "meet" at the barrier (and
    "reduce" its answer there), "look" at the flag."""
    body = re.search(r"bool quadrant_agrees\([^)]*\)\s*\{(.*?)\n\}", text, re.S).group(1)
    body = body.replace("quadrant_sync(quad);", "bar.sync;")
    marks = [(m.start(), s) for pattern, s in ((r"given_up\[[^\]]*\] = 1", "raise"), (r"bar\.sync", "meet"), (r"bar\.red\.and\.pred", "reduce"),
                                               (r"return given_up", "look")) for m in re.finditer(pattern, body)]
    return [s for _, s in sorted(marks)]


def _answers(steps, waits):
    """Every pair of answer lists that two warps can leave with, over all orders of their steps: each goes through the waits of its
    list until one gives up or the two of them do not agree."""
    flat = [(call, s) for call in range(len(waits[0])) for s in steps]
    ends, seen = set(), set()

    def go(at, met, joined, flag, answers):
        key = (at, met, joined, flag, answers)
        if key in seen:
            return
        seen.add(key)
        moved = False
        for w in (0, 1):
            if at[w] == len(flat) or answers[w][-1:] == (False,):
                continue
            call, step = flat[at[w]]
            m, j, f, a, n = met, joined, flag, answers, at[w] + 1
            if step in ("meet", "reduce"):
                if met[w] == call:                               # arrives
                    m = tuple(call + 1 if k == w else met[k] for k in (0, 1))
                    j = tuple(x and waits[w][c] if c == call else x for c, x in enumerate(joined))
                    n = at[w]
                elif met[1 - w] <= call:
                    continue                                     # waits for the other
                elif step == "reduce":
                    a = tuple(answers[k] + (joined[call],) if k == w else answers[k] for k in (0, 1))
            elif step == "raise":
                f = flag or not waits[w][call]
            else:
                a = tuple(answers[k] + (not flag,) if k == w else answers[k] for k in (0, 1))
            moved = True
            go(tuple(n if k == w else at[k] for k in (0, 1)), m, j, f, a)
        if not moved:
            ends.add(answers)

    go((0, 0), (0, 0), (True,) * len(waits[0]), False, ((), ()))
    return ends


@pytest.mark.parametrize("waits", [((True, True), (True, True)), ((False, True), (True, True)), ((True, True), (True, False)),
                                   ((True, True, False), (True, True, True)), ((True, False), (True, False))])
def test_two_warps_that_share_boxes_leave_together(waits):
    """Two warps share the boxes of a quadrant of the SwiGLU backward from codes and its barriers.  One that leaves while the
    other goes on would be waited for without end, so in every order of their steps both give the same answers."""
    steps = _agreement_steps(re.sub(r"//[^\n]*", "", (CSRC / "gemm_2sm.cu").read_text()))
    assert "meet" in steps or "reduce" in steps
    # the model tells a sound exchange from one whose flag is the next call's as well
    assert all(a == b for a, b in _answers(["reduce"], waits))
    for a, b in _answers(steps, waits):
        assert a == b, (steps, a, b)
    want = [all(w) for w in zip(*waits)]
    want = tuple(want[:want.index(False) + 1] if False in want else want)
    assert {a for a, _ in _answers(steps, waits)} == {want}


def test_the_model_of_two_warps_finds_a_flag_that_is_read_late():
    ends = _answers(["raise", "meet", "look"], ((True, True), (True, False)))
    assert any(a != b for a, b in ends)


@pytest.mark.parametrize("src", sorted(p.name for p in CSRC.glob("*.cu") if "extern __shared__" in p.read_text()))
def test_buffers_of_bytes_in_shared_memory_are_aligned_by_declaration_or_by_hand(src):
    """A dynamic buffer lies behind the kernel's static arrays.  One of bytes has no alignment of its own, and copies of 16 bytes
    fault on another: it is declared with one, or used through a pointer that was rounded up."""
    text = re.sub(r"//[^\n]*", "", (CSRC / src).read_text())
    for name, _, body in _kernels(src):
        for buf in re.findall(r"extern __shared__ (?:uint8_t|int8_t|char) (\w+)\[\];", body):
            uses = re.findall(rf"[^;]*\b{buf}\b[^;]*;", body.split(f"{buf}[];", 1)[1])
            assert uses and all(re.search(rf"\(reinterpret_cast<uintptr_t>\({buf}\) \+ \d+\) & ~", u) for u in uses), (name, buf)
    assert "extern __shared__" in text
