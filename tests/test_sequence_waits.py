"""The wait states around matrix instructions in the sequence-layer kernels that ship (CPU; needs the built library and ROCm's
llvm-objdump).  The compiler inserts them, but it does not look into inline assembly, and it has been seen to leave some out
behind branches:

    a vector instruction writes a register, a matrix instruction reads it    2 wait states between them
    a matrix instruction writes one, anything else reads or computes it      11 (10 behind fp32 products); a load's result
                                                                             arrives later, another product waits by itself

An instruction is one wait state, s_nop N is N + 1.  Every path through a kernel is followed, loops included."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "dsp_amd", "lib", "libdsp_gpu.so")
OBJDUMP = "/opt/rocm/lib/llvm/bin/llvm-objdump"
VECTOR, MATRIX = 2, {"v_mfma_f32_16x16x32_bf16": 11, "v_mfma_f32_16x16x4_f32": 10}

INSN = re.compile(r"^\s+(\S+)\s*(.*?)\s*//\s*([0-9A-Fa-f]+):")
TARGET = re.compile(r"<[^>]*\+0x([0-9a-fA-F]+)>\s*$")
REG = re.compile(r"\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])")


def registers(text):
    out = set()
    for kind, one, low, high in REG.findall(text):
        out.update(kind + str(i) for i in (range(int(one), int(one) + 1) if one else range(int(low), int(high) + 1)))
    return out


def kernels(text):
    """{name: [(address, mnemonic, operands, branch target)]}"""
    out, cur = {}, None
    for line in text.splitlines():
        head = re.match(r"^([0-9a-f]+) <(.+)>:$", line)
        if head:
            start, cur = int(head.group(1), 16), []
            if "linear_attention_kernel" in head.group(2):
                out[head.group(2)] = cur
            continue
        m = INSN.match(line)
        if m and cur is not None:
            t = TARGET.search(line) if m.group(1).startswith(("s_cbranch", "s_branch")) else None
            cur.append((int(m.group(3), 16), m.group(1), m.group(2), start + int(t.group(1), 16) if t else None))
    return out


def analyse(insns):
    """Places where a wait is short, and how many matrix instructions were looked at."""
    index = {a: i for i, (a, _, _, _) in enumerate(insns)}
    leaders = {0}
    for i, (_, op, _, to) in enumerate(insns):
        if to is not None:
            leaders.add(index[to])
        if to is not None or op == "s_endpgm":
            leaders.add(i + 1)
    order = sorted(x for x in leaders if x < len(insns))
    end = dict(zip(order, order[1:] + [len(insns)]))
    entry, work, errors, matrix = {0: {}}, [0], set(), 0

    def run(block, state, report):
        """state: (register, written by) -> wait states still missing"""
        state = dict(state)
        for i in range(block, end[block]):
            _, op, ops, _ = insns[i]
            parts = [p.strip() for p in ops.split(",")] if ops else []
            product, load = op.startswith("v_mfma"), bool(re.match(r"(ds_read|(buffer|global|scratch)_load)", op))
            if report and parts:
                if product:
                    bad = [r for r in registers(",".join(parts[1:4])) if (r, "vector") in state]
                else:
                    bad = [r for r in registers(",".join(parts[load:])) if (r, "matrix") in state]
                errors.update((hex(insns[i][0]), op, ops, r) for r in bad)
            passed = int(parts[0], 0) + 1 if op == "s_nop" else 1
            state = {k: n - passed for k, n in state.items() if n > passed}
            if product:
                for r in registers(",".join(parts[1:4])):
                    state.pop((r, "matrix"), None)
            if parts and (load or op.startswith("v_")):
                for r in registers(parts[0]):
                    state.pop((r, "matrix"), None)
                    state.pop((r, "vector"), None)
                    if not load:
                        state[(r, "matrix" if product else "vector")] = MATRIX[op] if product else VECTOR
        last = insns[end[block] - 1]
        after = [index[last[3]]] if last[3] is not None else []
        if last[1] not in ("s_branch", "s_endpgm") and end[block] < len(insns):
            after.append(end[block])
        return state, after

    while work:
        block = work.pop()
        state, after = run(block, entry[block], False)
        for b in after:
            old = entry.get(b)
            new = dict(old or {})
            for k, n in state.items():
                new[k] = max(n, new.get(k, n))
            if new != old:
                entry[b] = new
                work.append(b)
    for block, state in entry.items():
        run(block, state, True)
        matrix += sum(insns[i][1].startswith("v_mfma") for i in range(block, end[block]))
    return sorted(errors), matrix


def test_the_walk_sees_short_waits():
    """Planted in text: one wait state between a vector write and a product, ten behind a product, both across a loop's end."""
    def code(*lines):
        return [(4 * i, *(x + ("",) * (2 - len(x))), to) for i, (x, to) in enumerate(lines)]
    mfma, nop = ("v_mfma_f32_16x16x32_bf16", "v[0:3], v[4:7], v[8:11], v[0:3]"), ("s_nop", "9")
    assert analyse(code((("v_mul_f32", "v4, v20, v21"), None), (("s_nop", "0"), None), (mfma, None), (("s_endpgm",), None)))[0]
    assert not analyse(code((("v_mul_f32", "v4, v20, v21"), None), (("s_nop", "1"), None), (mfma, None), (("s_endpgm",), None)))[0]
    assert analyse(code((mfma, None), (nop, None), (("v_mul_f32", "v20, v1, v21"), None), (("s_endpgm",), None)))[0]
    assert not analyse(code((mfma, None), (("s_nop", "10"), None), (("v_mul_f32", "v20, v1, v21"), None), (("s_endpgm",), None)))[0]
    assert analyse(code((mfma, None), (("v_mul_f32", "v9, v20, v21"), None), (("s_cbranch_scc1", ""), 0), (("s_endpgm",), None)))[0]


@pytest.mark.parametrize("sample", ["DF16bDF16b", "DF16_f", "ff"], ids=["bf16", "fp16", "fp32"])
def test_waits_around_matrix_instructions(tmp_path, sample):
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("needs dsp_amd/lib/libdsp_gpu.so and llvm-objdump")
    local = shutil.copy(LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", local], check=True, cwd=tmp_path, capture_output=True)
    seen = 0
    for f in sorted(os.listdir(tmp_path)):
        path = tmp_path / f
        if "gfx950" not in f or f"linear_attention_kernelI{sample}" not in subprocess.run([OBJDUMP, "-t", path], check=True, capture_output=True, text=True).stdout:
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout
        for name, insns in kernels(text).items():
            errors, matrix = analyse(insns)
            assert not errors, (name, len(errors), errors[:5])
            assert matrix > 20, name
            seen += 1
    assert seen == 20  # five shapes, with and without outputs, with and without whole packs
