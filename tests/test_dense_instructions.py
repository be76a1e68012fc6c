"""The large tiles of the dense layers write their matrix instructions as inline assembly, whose hazards the compiler does not see.  What its output has to hold is checked on the built library, so
that another compiler version, or a change beside them, that breaks it is found here:
  - no vector instruction writes an operand of a matrix instruction in the two wait states before it,
  - nothing but a matrix instruction touches its sums in the 19 wait states behind it (the longest that a matrix instruction of up to 16 passes asks for),
  - its factors are vector registers, its sums accumulation registers (so none waits for another's result but its own),
  - M0 is written in front of a load to LDS and named nowhere else,
and for all of the dense layers and clipping: no packed 32-bit floating point instruction."""
import os
import re
import shutil
import subprocess

import pytest

import ngp_abi as A

TOOLS = "/opt/rocm/llvm/bin"
WRITE_WAIT, READ_WAIT = 2, 19


def registers(text):
    """{('v' | 'a', number)} of a list of operands"""
    out = set()
    for kind, first, last, one in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out |= {(kind, r) for r in (range(int(first), int(last) + 1) if first else [int(one)])}
    return out


def parse(lines):
    """[(address, instruction, operands)] of one function's listing"""
    code = []
    for line in lines:
        m = re.match(r"\s+(\S+)\s*(.*?)\s*//\s*([0-9A-Fa-f]+):", line)
        if m:
            code.append((int(m[3], 16), m[1], m[2]))
    return code


def flow(code):
    """successors of every instruction"""
    at = {a: i for i, (a, *_) in enumerate(code)}
    after = []
    for i, (a, name, ops) in enumerate(code):
        nexts = [] if name in ("s_endpgm", "s_branch", "s_setpc_b64") else [i + 1] if i + 1 < len(code) else []
        if name == "s_branch" or name.startswith("s_cbranch"):
            offset = int(ops.split()[0])
            target = a + 4 + 4 * (offset - 65536 if offset > 32767 else offset)
            assert target in at, "a branch out of the function"
            nexts.append(at[target])
        assert name != "s_setpc_b64", "an indirect jump"
        after.append(nexts)
    return after


def waits(name, ops):
    return int(ops, 0) + 1 if name == "s_nop" else 1


def hazards(code):
    """what is wrong in a function, as text"""
    after = flow(code)
    before = [[] for _ in code]
    for i, n in enumerate(after):
        for j in n:
            before[j].append(i)
    bad, count = [], 0

    def walk(i, edges, limit, look):
        """every instruction within `limit` wait states of i along the edges"""
        seen, todo = {}, [(j, 0) for j in edges[i]]
        while todo:
            j, passed = todo.pop()
            if passed >= limit or seen.get(j, limit) <= passed:
                continue
            seen[j] = passed
            look(j)
            passed += waits(code[j][1], code[j][2])
            todo += [(k, passed) for k in edges[j]]

    for i, (address, name, ops) in enumerate(code):
        if not name.startswith("v_mfma"):
            if "m0" in re.split(r"[\s,]+", ops):
                follow = [c[1] for c in code[i + 1:i + 3]]
                if name != "s_mov_b32" or follow[:1] != ["s_nop"] or not follow[1].startswith("buffer_load") or "lds" not in code[i + 2][2]:
                    bad.append(f"{address:x}: M0 in {name} {ops}")
            continue
        count += 1
        sums, *factors = [registers(o) for o in re.split(r",\s*(?![^\[]*\])", ops)][:3]
        carry = registers(re.split(r",\s*(?![^\[]*\])", ops)[3])
        if carry != sums or any(k != "a" for k, _ in sums) or any(k != "v" for f in factors for k, _ in f):
            bad.append(f"{address:x}: registers of {name} {ops}")
        reads = sums.union(*factors)

        def writes_operand(j):
            n, o = code[j][1], code[j][2]
            if n.startswith("v_") and not n.startswith(("v_mfma", "v_cmp")) and registers(o.split(",")[0]) & reads:
                bad.append(f"{address:x}: {name} {ops} closely behind {n} {o}")

        def touches_sums(j):
            n, o = code[j][1], code[j][2]
            if not n.startswith("v_mfma") and registers(o) & sums:
                bad.append(f"{address:x}: {n} {o} closely behind {name} {ops}")
        walk(i, before, WRITE_WAIT, writes_operand)
        walk(i, after, READ_WAIT, touches_sums)
    return bad, count


def listing(text):
    return parse([f"\t{line} // {4 * i:012X}: 00000000" for i, line in enumerate(text)])


MFMA = "v_mfma_f32_16x16x32_f16 a[0:3], v[0:3], v[4:7], a[0:3]"


@pytest.mark.parametrize("text,wrong", [
    (["ds_read_b128 v[0:3], v9", "s_waitcnt lgkmcnt(0)", MFMA, "s_nop 15", "s_nop 15", "v_accvgpr_read_b32 v0, a0", "s_endpgm"], 0),
    (["v_mov_b32_e32 v3, v9", "s_nop 0", MFMA, "s_endpgm"], 1),
    (["v_mov_b32_e32 v3, v9", "s_nop 1", MFMA, "s_endpgm"], 0),
    (["v_accvgpr_write_b32 a2, 0", MFMA, "s_endpgm"], 1),
    ([MFMA, "s_nop 15", "v_accvgpr_read_b32 v0, a3", "s_endpgm"], 1),
    ([MFMA, "s_nop 15", "ds_write_b128 v9, a[0:3]", "s_endpgm"], 1),
    ([MFMA, MFMA, "s_nop 15", "s_nop 2", "v_accvgpr_read_b32 v0, a3", "s_endpgm"], 0),
    (["s_nop 3", MFMA, "v_add_u32_e32 v5, 1, v5", "s_cbranch_scc1 65533", "s_endpgm"], 1),      # back to the matrix instruction
    ([MFMA, "s_cbranch_scc1 2", "s_nop 15", "s_nop 15", "v_accvgpr_read_b32 v0, a3", "s_endpgm"], 1),  # past the waits
    (["v_mfma_f32_16x16x32_f16 v[0:3], v[0:3], v[4:7], v[0:3]", "s_endpgm"], 1),
    (["s_mov_b32 m0, s3", "s_nop 0", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds", "s_endpgm"], 0),
    (["s_mov_b32 m0, s3", "s_add_u32 s1, s1, m0", "s_endpgm"], 2),
])
def test_the_check_itself(text, wrong):
    assert len(hazards(listing(text))[0]) == wrong


@pytest.fixture(scope="module")
def code_objects(tmp_path_factory):
    """the library's device code, one file per source file"""
    if not os.path.exists(os.path.join(TOOLS, "llvm-objdump")):
        pytest.skip("no llvm-objdump")
    d = tmp_path_factory.mktemp("code")
    lib = shutil.copy(A.LIB_PATH, d)
    subprocess.run([os.path.join(TOOLS, "llvm-objdump"), "--offloading", os.path.basename(lib)], cwd=d, check=True, capture_output=True)
    out = {}
    for f in sorted(d.iterdir()):
        if "gfx950" in f.name:
            table = subprocess.run([os.path.join(TOOLS, "llvm-objdump"), "-t", str(f)], check=True, capture_output=True, text=True).stdout
            out[str(f)] = re.findall(r" F \.text\s+[0-9a-f]+ (?:\.\w+ )?(\S+)$", table, re.M)
    return out


def test_matrix_instructions_in_place(code_objects):
    checked = matrix = 0
    for path, symbols in code_objects.items():
        names = [s for s in symbols if re.search(r"k_(gemm|products)_async", s)]
        if not names:
            continue
        p = subprocess.Popen([os.path.join(TOOLS, "llvm-objdump"), "-d", "--no-show-raw-insn", "--disassemble-symbols=" + ",".join(names), path], stdout=subprocess.PIPE, text=True)
        function, lines = None, []
        for line in [*p.stdout, "0 <end>:"]:
            if re.match(r"[0-9a-f]+ <.*>:", line):
                if function:
                    bad, count = hazards(parse(lines))
                    assert not bad, (function, len(bad), bad[:5])
                    checked, matrix = checked + 1, matrix + count
                function, lines = line, []
            else:
                lines.append(line)
        assert p.wait() == 0
    assert checked >= 20 and matrix >= 32 * checked  # (both element types)


def test_no_packed_floats(code_objects):
    checked = 0
    for path, symbols in code_objects.items():
        if any(re.search(r"k_gemm_async|k_clip_small", s) for s in symbols):
            p = subprocess.Popen([os.path.join(TOOLS, "llvm-objdump"), "-d", "--no-show-raw-insn", path], stdout=subprocess.PIPE, text=True)
            found = [line for line in p.stdout if re.search(r"\bv_pk_(add|mul|fma)_f32\b", line)]
            assert p.wait() == 0 and not found, (path, found[:3])
            checked += 1
    assert checked == 3


def test_no_packed_floats_in_any_kernel(code_objects):
    """all of the library is compiled without them"""
    found = {}
    for path, symbols in code_objects.items():
        p = subprocess.Popen([os.path.join(TOOLS, "llvm-objdump"), "-d", "--no-show-raw-insn", path], stdout=subprocess.PIPE, text=True)
        n = sum("v_pk_" in line and re.search(r"\bv_pk_(add|mul|fma)_f32\b", line) is not None for line in p.stdout)
        assert p.wait() == 0
        if n:
            found[os.path.basename(path)] = n
    assert len(code_objects) >= 9 and not found, found
