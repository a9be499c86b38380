"""The products of the orthogonalised updates wait for LDS-DMA by count, with a known number of other loads in flight (mu_mainloop in
muon.hip): too few of those, as after a merge of two by the compiler, and a wait lets a stage be read before it has landed.  So the
built library's own instructions are counted."""
import os
import re
import shutil
import subprocess

import pytest

from mdnvae_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
RING = 5                                                     # stages, MU_RING


def kernels(tmp_path):
    """{demangled name: [(instruction, operands)]} of the tiled products in the built library."""
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found = {}
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name or b"mu_step_kernel" not in (tmp_path / name).read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--demangle", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        body = None
        for line in text.splitlines():
            head = re.match(r"^[0-9a-f]+ <(?:void )?mdnvae::(mu_(?:step|sym)_kernel<[^>]*>)", line)
            if head:
                body = found.setdefault(head.group(1), [])
            elif re.match(r"^[0-9a-f]+ <", line):
                body = None
            elif body is not None:
                op = re.match(r"^\s+([a-z]\w+)\s*([^/]*)", line)
                if op:
                    body.append((op.group(1), op.group(2).strip()))
    return found


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_loads_beside_the_dmas_are_as_many_as_the_waits_count_on(tmp_path):
    found = kernels(tmp_path)
    seen = 0
    for name, body in found.items():
        args = [a.strip() for a in name[name.index("<") + 1:-1].split(",")]
        step = name.startswith("mu_step")
        tile, terms = (int(v) for v in (args[2:4] if step else args[1:3]))
        parts, blocks = 2 if terms == 3 else 1, (tile // 64) ** 2
        pieces = tile // 32 * parts // 2                     # DMAs of a stage and wave
        assert not any(op.startswith(("scratch_", "buffer_")) for op, _ in body), name      # spills would move the count
        if step:
            extra = blocks * 8                               # both parts of X
        elif args[3] == "1":
            extra = blocks * 4 * parts                       # A, as many parts as there are terms
        else:
            extra = 0
        counted = [i for i, (op, arg) in enumerate(body) if op == "s_waitcnt" and f"vmcnt({(RING - 3) * pieces + extra})" in arg
                   and body[i + 1][0] == "s_barrier"]
        if not extra:
            assert counted and not any(op == "global_load_dwordx2" for op, _ in body[counted[0]:]), name
            continue
        # three steps run with the loads in flight; they were issued since the last barrier ahead of the first of them
        assert len(counted) == 3, (name, len(counted))
        assert (RING - 3) * pieces + extra < 64, name
        last = max(i for i in range(counted[0]) if body[i][0] == "s_barrier")
        between = [op for op, _ in body[last:counted[0]] if op.startswith(("global_load", "global_store", "global_atomic", "flat_"))]
        assert between.count("global_load_dwordx2") == extra, (name, between.count("global_load_dwordx2"))
        assert between.count("global_load_lds_dwordx4") == len(between) - extra, (name, between)
        # and between the counted waits a stage's DMAs alone
        for a, b in zip(counted, counted[1:]):
            ops = [op for op, _ in body[a:b] if op.startswith(("global_", "flat_"))]
            assert ops == ["global_load_lds_dwordx4"] * pieces, (name, ops)
        seen += 1
    # one shape or a table; both types; two tiles; one or three terms; the last step or not; and B
    assert seen == 2 * 2 * 2 * 2 * 2 + 2 * 2 * 2
