"""What the compiler makes of kernels whose results or safety hang on it, read from listings of the library's own code (no GPU needed)."""
import collections
import os
import re
import shutil
import subprocess

import pytest

from hortimapping_amd import build as hb

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
pytestmark = pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")


def kernel(listing, name):
    """Body of the one kernel whose mangled name holds `name`."""
    starts = [m for m in re.finditer(r"^(_Z\S+):", listing, re.M) if name in m[1]]
    assert len(starts) == 1, [m[1] for m in starts]
    body = listing[starts[0].end():]
    return body[:body.index(".Lfunc_end")]


def test_transformed_points_do_not_hang_on_the_compilers_choice(tmp_path):
    """The sums of products of both point transforms round the same way whether the compiler may fuse products into sums across
    statements (its default here), within one, or not at all: all fusing is written out."""
    modes = ("fast-honor-pragmas", "on", "off")
    count = {}
    for contract in modes:
        out = str(tmp_path / f"{contract}.s")
        subprocess.run([HIPCC] + hb.FLAGS + [f"-ffp-contract={contract}", "-S", "--cuda-device-only", os.path.join(hb.CSRC, "hm_render.hip"),
                                             "-o", out], check=True, capture_output=True)
        listing = open(out).read()
        for name in ("k_transform_points", "k_sample_rays"):
            count[name, contract] = collections.Counter(re.findall(r"^\s+(v_(?:fma|mul|add|sub)\w*_f32)", kernel(listing, name), re.M))
    for name in ("k_transform_points", "k_sample_rays"):
        assert count[name, modes[0]] == count[name, "on"] == count[name, "off"] and sum(count[name, "off"].values()) >= 13


# ---- the wide projection names its accumulation registers itself, so the compiler neither keeps them free nor waits for them

OBJDUMP, READOBJ = (os.path.join("/opt/rocm/llvm/bin", n) for n in ("llvm-objdump", "llvm-readobj"))


class Code:
    """One kernel: instructions as (mnemonic, operands), and where control may come from."""

    def __init__(self, lines):
        self.ins, self.before, at, jumps = [], [], {}, []
        for line in lines:
            m = re.match(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):.*?(?:<\S+\+0x([0-9a-f]+)>)?$", line)
            if m is None:
                continue
            i = len(self.ins)
            at[int(m[3], 16)] = i
            self.ins.append((m[1], [o.strip() for o in m[2].split(",")] if m[2] else []))
            if m[4] is not None and m[1].startswith(("s_branch", "s_cbranch")):
                jumps.append((i, int(m[4], 16)))
        start = min(at)
        self.before = [[i - 1] if i > 0 and self.ins[i - 1][0] not in ("s_branch", "s_endpgm") else [] for i in range(len(self.ins))]
        for i, offset in jumps:
            self.before[at[start + offset]].append(i)

    def back(self, i, states):
        """Instructions that may have run within `states` wait states before instruction i."""
        seen, todo = {}, [(j, states) for j in self.before[i]]
        while todo:
            j, left = todo.pop()
            if left <= 0 or seen.get(j, 0) >= left:
                continue
            seen[j] = left
            op, args = self.ins[j]
            left -= int(args[0]) + 1 if op == "s_nop" else 1
            todo += [(p, left) for p in self.before[j]]
        return seen


def registers(operand, kind):
    m = re.fullmatch(kind + r"(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if m is None:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


@pytest.fixture(scope="module")
def wide(tmp_path_factory):
    """({name: Code}, metadata) of the wide projection's kernels in the built library."""
    if not os.path.exists(hb.LIB):
        hb.build(verbose=False)
    if not (os.path.exists(OBJDUMP) and os.path.exists(READOBJ)):
        pytest.skip("no llvm-objdump")
    td = str(tmp_path_factory.mktemp("lib"))
    shutil.copy(hb.LIB, os.path.join(td, "lib.so"))
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=td, check=True, capture_output=True)
    run = lambda *a: subprocess.run(a, cwd=td, check=True, capture_output=True, text=True).stdout  # noqa: E731
    files = [f for f in os.listdir(td) if f.endswith("gfx950") and "k_project_wide" in run(OBJDUMP, "-t", f)]
    assert len(files) == 1
    code, name = {}, None
    for line in run(OBJDUMP, "-d", "--mcpu=gfx950", files[0]).split("\n"):
        m = re.match(r"[0-9a-f]{16} <(\S+)>:", line)
        if m:
            name = m[1]
        elif name is not None and "k_project_wide" in name:
            code.setdefault(name, []).append(line)
    assert len(code) == 6                               # three types, with and without a mask
    return {n: Code(lines) for n, lines in code.items()}, run(READOBJ, "--notes", files[0])


def test_nothing_else_touches_the_sums_of_the_wide_projection(wide):
    kernels, notes = wide
    for name, code in kernels.items():
        count = collections.Counter()
        for op, args in code.ins:
            if not any(registers(a, "a") for a in args):
                continue
            if op.startswith("v_mfma"):                 # a sum is added to where it is, of operands in ordinary registers
                assert args[0] == args[3] and len(registers(args[0], "a")) == 16 and registers(args[1], "v") and registers(args[2], "v"), (name, op, args)
            elif op == "v_accvgpr_write_b32":
                assert args[1] == "0", (name, args)     # cleared, nothing else
            else:
                assert op == "v_accvgpr_read_b32", (name, op, args)
            count[op] += 1
        assert count["v_accvgpr_write_b32"] == 256 and count["v_accvgpr_read_b32"] == 256, (name, count)
        assert not any(op.startswith("scratch_") for op, _ in code.ins), name
        entry = notes[:notes.index(name + ".kd")].rindex(".agpr_count")
        entry = notes[entry:notes.index(".wavefront_size", entry)]
        assert re.search(r"\.private_segment_fixed_size: 0\b", entry) and re.search(r"\.vgpr_spill_count: 0\b", entry), name


def test_products_of_the_wide_projection_wait_for_their_operands(wide):
    """Two wait states between a vector instruction and the product that reads what it wrote; a product between two on the same sum;
    eighteen states (sixteen passes of the longest product, and two) before a sum is read."""
    for name, code in wide[0].items():
        last = None
        for i, (op, args) in enumerate(code.ins):
            if op.startswith("v_mfma"):
                reads = registers(args[1], "v") | registers(args[2], "v") | registers(args[3], "v")
                for j in code.back(i, 2):
                    o, a = code.ins[j]
                    assert not (o.startswith("v_") and not o.startswith("v_mfma") and registers(a[0], "v") & reads), (name, o, a, op, args)
                if registers(args[0], "a"):
                    assert last != args[0], (name, op, args)
                    last = args[0]
            elif op == "v_accvgpr_read_b32":
                assert not any(code.ins[j][0].startswith("v_mfma") and registers(code.ins[j][1][0], "a") for j in code.back(i, 18)), (name, i)
