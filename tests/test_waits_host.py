"""The waits of linear_fp8's tile kernels in the library as it is built (CPU).

Between two barriers a wave of these kernels loads a step's data into LDS and
some scales into registers, and waits by counting loads: a compiler that loaded
fewer scales than the count assumes, or moved them, would leave data of the step
to be read in flight. So the kernels' own instructions are followed here along
every path: at a barrier no more loads into LDS may be under way than those of
the steps behind the next one."""
import functools
import os
import re
import shutil
import subprocess

import pytest

from dfsattn_amd import build

TOOL = "/opt/rocm/llvm/bin/llvm-objdump"
KERNEL = re.compile(r"fp8_tile_kernelILi(\d)ELi(\d)ELi(\d)ELi(\d)ELi(\d)ELb(\d)E")
pytestmark = pytest.mark.skipif(not os.path.exists(TOOL), reason="no llvm-objdump")


@functools.lru_cache(maxsize=None)
def _kernels():
    """{template arguments: [(address, instruction)]} of the tile kernels, up to their ends."""
    import tempfile

    found = {}
    with tempfile.TemporaryDirectory() as tmp:
        lib = shutil.copy(os.path.join(build.OUT_DIR, build.LIB_NAME), tmp)
        subprocess.run([TOOL, "--offloading", lib], cwd=tmp, check=True, capture_output=True)
        for name in sorted(os.listdir(tmp)):
            path = os.path.join(tmp, name)
            if "amdgcn" not in name or "fp8_tile_kernel" not in subprocess.run(
                    [TOOL, "-t", path], check=True, capture_output=True, text=True).stdout:
                continue
            text = subprocess.run([TOOL, "-d", path], check=True, capture_output=True, text=True).stdout
            at = None
            for line in text.splitlines():
                head = re.match(r"[0-9a-f]+ <(.*)>:", line)
                if head:
                    m = KERNEL.search(head.group(1))
                    at = found.setdefault(tuple(int(g) for g in m.groups()), []) if m else None
                elif at is not None and "// " in line:
                    op, _, comment = line.partition("// ")
                    at.append((int(comment.split(":")[0], 16), op.strip()))
    return found


def _most_under_way(code):
    """(most loads into LDS under way at the first barrier, at any later one) over all paths."""
    index = {a: i for i, (a, _) in enumerate(code)}

    def after(i):
        address, op = code[i]
        word = op.split()[0]
        if word == "s_endpgm":
            return ()
        if word == "s_branch" or word.startswith("s_cbranch"):
            n = int(op.split()[1])
            target = index[address + 4 + 4 * (n - 0x10000 if n >= 0x8000 else n)]
            return (target,) if word == "s_branch" else (i + 1, target)
        assert not word.startswith(("s_setpc", "s_swappc")), op
        return (i + 1,)

    def into_lds(op):
        return op.startswith("buffer_load") and op.endswith(" lds")

    # what lies behind the last load into LDS is not followed
    before = [[] for _ in code]
    for i in range(len(code)):
        for j in after(i):
            if j < len(code):  # behind the last branch lies padding
                before[j].append(i)
    alive, todo = set(), [i for i, (_, op) in enumerate(code) if into_lds(op) or op == "s_barrier"]
    while todo:
        i = todo.pop()
        if i not in alive:
            alive.add(i)
            todo += before[i]
    most, seen, todo = [0, 0], set(), [(0, "", False)]
    while todo:
        state = todo.pop()
        i, queue, passed = state
        if i not in alive or state in seen:
            continue
        seen.add(state)
        op = code[i][1]
        if op.startswith("s_waitcnt"):
            m = re.search(r"vmcnt\((\d+)\)", op)
            if m:
                n = int(m.group(1))
                queue = queue[len(queue) - n:] if n < len(queue) else queue
        elif op == "s_barrier":
            most[passed] = max(most[passed], queue.count("d"))
            passed = True
        elif into_lds(op):
            queue += "d"
        elif re.match(r"(global|buffer|flat|scratch)_", op):
            queue += "s"
        assert len(queue) < 64 and len(seen) < 10 ** 6
        todo += [(j, queue, passed) for j in after(i)]
    return tuple(most)


def _allowed(kernel):
    ni, mi, wn, wm, buffers, _ = kernel
    data = ni * wn + mi * wm  # loads of a wave and step
    return (buffers - 1) * data, (buffers - 2) * data


def test_every_tile_kernel_is_there():
    assert {k[:5] for k in _kernels()} == {(1, 1, 2, 2, 4), (1, 2, 2, 2, 3), (2, 2, 2, 2, 3), (2, 2, 2, 2, 2)}
    assert len(_kernels()) == 8


@pytest.mark.parametrize("n", range(8))
def test_data_has_landed_at_each_barrier(n):
    kernel = sorted(_kernels())[n]
    first, later = _most_under_way(_kernels()[kernel])
    most = _allowed(kernel)
    assert 0 < first <= most[0] and 0 <= later <= most[1], kernel


@pytest.mark.parametrize("n", range(8))
def test_a_load_fewer_is_seen(n):
    """The same instructions without one of a step's loads of scales fail the check."""
    kernel = sorted(_kernels())[n]
    code = _kernels()[kernel]
    barriers = [i for i, (_, op) in enumerate(code) if op == "s_barrier"]
    scales = [i for i in range(barriers[0], barriers[-1]) if code[i][1].startswith("global_load_ubyte")]
    assert scales
    i = scales[-1]
    changed = code[:i] + [(code[i][0], "s_nop 0")] + code[i + 1:]
    assert _most_under_way(changed)[1] > _allowed(kernel)[1]
