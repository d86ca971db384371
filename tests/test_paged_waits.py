"""CPU check of the built code of the paged attention: wait states that the
hardware does not enforce, and that the compiler does not see to where inline
asm is on either side (it fills them in for its own instructions only), are
there on every path.

  - a buffer load reads a scalar register five wait states or more after a
    vector instruction (a lane read) wrote it: behind fewer it may take the old
    value, here the size that bounds the load;
  - the result of a matrix product is read by another kind of instruction its
    passes and four wait states later: behind fewer it is the value before.

Disassembles the kernels of this library only, and follows every branch."""
import os
import re
import shutil
import subprocess

import pytest

from ter_amd import _lib as L

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
SGPR_WAIT = 5
# passes of four cycles a SIMD needs for one (others: the most there are)
PASSES = {"v_mfma_f32_32x32x16_f16": 8, "v_mfma_f32_32x32x16_bf16": 8, "v_mfma_f32_16x16x32_f16": 4,
          "v_mfma_f32_16x16x32_bf16": 4, "v_mfma_f32_16x16x16_f16": 4, "v_mfma_f32_16x16x16_bf16": 4}


def registers(text):
    out = set()
    for kind, one, first, last in re.findall(r"(?<!\w)([vsa])(?:(\d+)|\[(\d+):(\d+)\])", text):
        out |= {kind + one} if one else {f"{kind}{i}" for i in range(int(first), int(last) + 1)}
    return out


def operands(op, args):
    """Registers that an instruction writes and reads (of a matrix product
    without the sums it adds to, which the matrix cores hand on themselves)."""
    parts = args.split(",")
    rest = ",".join(parts[1:])
    if op.startswith("v_mfma"):
        return registers(parts[0]), registers(",".join(parts[1:3]))
    if op.startswith("v_"):
        if "swap" in op:
            return registers(args), registers(args)
        own = registers(parts[0]) if re.search("writelane|dpp|fmac|dot2c", op) else set()
        return registers(parts[0]), registers(rest) | own
    if op.startswith(("buffer_", "global_", "flat_", "scratch_", "ds_")):
        if re.search("load|read", op) and " lds" not in args:
            return registers(parts[0]), registers(rest)
        return set(), registers(args)
    return set(), set()


def is_memory(op):
    return op.startswith(("buffer_", "global_", "flat_", "scratch_"))


class Kernel:
    def __init__(self, code):
        """code: (address, mnemonic, operands) of each instruction."""
        self.code = code
        at = {a: i for i, (a, _, _) in enumerate(code)}
        self.next = []
        for i, (a, op, args) in enumerate(code):
            to = [] if op in ("s_endpgm", "s_branch") else [i + 1]
            if op.startswith(("s_branch", "s_cbranch")):
                by = int(args.split()[0])
                to.append(at[a + 4 + 4 * (by - 65536 if by >= 32768 else by)])
            self.next.append([s for s in to if s < len(code)])

    def faults(self):
        """Instructions that some path reaches too early."""
        open_at = [None] * len(self.code)  # register -> wait states still to pass, the most of any path
        open_at[0] = {}
        work = [0]
        while work:
            i = work.pop()
            _, op, args = self.code[i]
            wait = int(args) + 1 if op == "s_nop" else 1
            now = {r: n - wait for r, n in open_at[i].items() if n > wait}
            writes, _ = operands(op, args)
            if op.startswith("v_mfma"):
                now.update({r: PASSES.get(op, 16) + 4 for r in writes})
            elif op.startswith("v_"):
                now = {r: n for r, n in now.items() if r not in writes}
                now.update({r: SGPR_WAIT for r in writes if r[0] == "s"})
            for s in self.next[i]:
                if open_at[s] is None:
                    open_at[s] = dict(now)
                elif any(open_at[s].get(r, 0) < n for r, n in now.items()):
                    open_at[s] = {r: max(open_at[s].get(r, 0), now.get(r, 0)) for r in {*open_at[s], *now}}
                else:
                    continue
                work.append(s)
        out = []
        for (a, op, args), left in zip(self.code, open_at):
            if left is None or op.startswith("v_mfma"):
                continue
            writes, reads = operands(op, args)
            early = {r: n for r, n in left.items() if r in reads and (r[0] != "s" or is_memory(op))}
            early.update({r: n for r, n in left.items() if r in writes and r[0] != "s" and op.startswith("v_")})
            if early:
                out.append(f"{op} {args}: {early}")
        return out


def kernels(tmp_path, name):
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump not installed")
    lib = shutil.copy(L.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    found = {}
    for f in sorted(tmp_path.iterdir()):
        if "gfx950" not in f.name or name.encode() not in f.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True, stdout=subprocess.PIPE,
                              text=True).stdout
        code = None
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(\S+)>:", line)
            if head:
                code = found.setdefault(head.group(1), []) if name in head.group(1) else None
                continue
            m = re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
            if m and code is not None:
                code.append((int(m.group(3), 16), m.group(1), m.group(2)))
    return {n: Kernel(c) for n, c in found.items()}


def test_the_check_itself():
    """Planted in the oracle's input: too early, in time, too early on one path only."""
    def faults(*lines):
        return len(Kernel([(4 * i, *l.split(" ", 1)) if " " in l else (4 * i, l, "") for i, l in enumerate(lines)]).faults())

    lane, load, end = "v_readlane_b32 s6, v1, 0", "buffer_load_dwordx4 v2, s[4:7], 0 offen lds", "s_endpgm"
    assert faults(lane, "s_nop 3", load, end) == 1
    assert faults(lane, "s_nop 4", load, end) == 0
    assert faults(lane, "s_mov_b32 m0, s9", "s_nop 3", load, end) == 0
    assert faults(lane, "s_cbranch_scc0 1", "s_nop 7", load, end) == 1
    mma = "v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], v[0:15]"
    assert faults(mma, "s_nop 7", "s_nop 2", "v_mul_f32_e32 v3, v3, v40", end) == 1
    assert faults(mma, "s_nop 7", "s_nop 3", "v_mul_f32_e32 v3, v3, v40", end) == 0
    assert faults(mma, "v_mov_b32_e32 v3, 0", end) == 1
    assert faults(mma, mma, "s_nop 7", "s_nop 3", "global_store_dword v50, v3, s[0:1]", end) == 0


def test_registers_suffice(tmp_path):
    """No scratch memory in the attention kernels: it is one more wait for all
    loads in flight, and memory for every wave."""
    for name, k in kernels(tmp_path, "paged_attend_kernel").items():
        assert not any(op.startswith("scratch_") for _, op, _ in k.code), name


def test_wait_states(tmp_path):
    found = kernels(tmp_path, "paged_attend_kernel")
    assert len(found) == 4
    for name, k in found.items():
        assert sum(op.startswith("v_mfma") for _, op, _ in k.code) >= 32, name
        assert sum(" lds" in args for _, _, args in k.code) >= 12, name
        bad = k.faults()
        assert not bad, (name, bad[:5])
