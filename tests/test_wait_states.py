"""What the compiler made of the kernels for microscaled rows: between a scaled matrix product and the first other instruction that touches its result there are the wait
states that the result takes.  Registers are followed along every way through the code."""
import os
import re
import subprocess

import pytest

from test_kernel_resources import _code_objects
from vtl_amd import capi

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
REGISTERS = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operands):
    """The vector and accumulation registers that are named."""
    found = set()
    for kind, first, last, one in REGISTERS.findall(operands):
        found |= {(kind, n) for n in (range(int(first), int(last) + 1) if first else [int(one)])}
    return found


def needed(text):
    """Wait states behind a scaled product: a pass is four cycles; three more, and one on this chip.  16x16x128 takes four passes, and 32x32x64 eight, twice as many where an
    operand is of 8 bits (cbsz and blgp 4: 4 bits)."""
    passes = 4 if "16x16x128" in text else 8
    if "cbsz:4" not in text or "blgp:4" not in text:
        passes *= 2
    return passes + 4


class Function:
    def __init__(self, lines):
        self.text, self.next = [], []
        at = {}
        for line in lines:
            code, _, rest = line.partition("//")
            self.text.append(code.strip())
            at[int(rest.split(":")[0], 16)] = len(self.text) - 1
        places = sorted(at)
        for address in places:
            i, code = at[address], self.text[at[address]]
            follow = [] if re.match(r"s_endpgm|s_branch", code) else [i + 1] if i + 1 < len(self.text) else []
            jump = re.match(r"s_c?branch\w* (\d+)", code)
            if jump:
                words = int(jump[1])
                target = address + 4 + 4 * (words - 65536 if words >= 32768 else words)
                follow.append(at[target])
            assert not re.match(r"s_(setpc|swappc|call)", code), code
            self.next.append(follow)

    def too_early(self):
        """(the product, what touches its result, the wait states between them, those that it takes) where there are fewer, and the least that there are anywhere."""
        bad, least = [], 99
        for i, code in enumerate(self.text):
            if not code.startswith("v_mfma_scale"):
                continue
            result, enough = registers(code.split(",")[0]), needed(code)
            best, queue = {}, [(j, 0) for j in self.next[i]]
            while queue:
                j, states = queue.pop()
                if states > enough or best.get(j, 99) <= states:
                    continue
                best[j] = states
                other = self.text[j]
                if other.startswith("v_mfma"):
                    operands = other.split(None, 1)[1].split(", ")
                    if registers(" ".join(operands[1:3])) & result:
                        bad.append((code, other, states, enough))
                    if registers(operands[0]) & result:
                        continue        # takes it up as it is, and has a result of its own
                elif registers(other) & result:
                    least = min(least, states - enough)
                    if states < enough:
                        bad.append((code, other, states, enough))
                    continue
                nop = re.match(r"s_nop (\d+)", other)
                queue += [(k, states + (int(nop[1]) + 1 if nop else 1)) for k in self.next[j]]
        return bad, least


def functions(text):
    lines = None
    for line in text.splitlines():
        if re.match(r"[0-9a-f]+ <(.*)>:$", line):
            lines = []
            yield re.match(r"[0-9a-f]+ <(.*)>:$", line)[1], lines
        elif lines is not None and line.startswith("\t") and "//" in line:
            lines.append(line)


def disassembled(path):
    text = subprocess.run([OBJDUMP, "-d", str(path)], stdout=subprocess.PIPE, text=True, check=True).stdout
    return [(name, lines) for name, lines in list(functions(text)) if "mxfp4" in name or "moe" in name]


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs llvm-objdump")
def test_results_of_products_are_waited_for(tmp_path):
    with_products, bad, close = 0, [], []
    for i, code in enumerate(_code_objects(open(capi.LIB_PATH, "rb").read())):
        path = tmp_path / f"{i}.o"
        path.write_bytes(code)
        if b"mxfp4" not in code and b"moe_" not in code:
            continue
        for name, lines in disassembled(path):
            f = Function(lines)
            with_products += any(t.startswith("v_mfma_scale") for t in f.text)
            early, least = f.too_early()
            bad += [(name, *b) for b in early]
            # written in the source in front of whatever comes first, copies from accumulation registers among it
            close += [(name, least)] * (least < 1)
    assert with_products > 20 and not bad, (with_products, bad[:4])
    assert not close, close


def test_a_read_on_the_shorter_of_two_ways_is_found():
    product = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[0:3], v[4:11], a[0:3], v12, v13 op_sel_hi:[0,0,0] cbsz:4"
    code = [product, "s_cbranch_execz 2", "s_nop 6", "s_nop 0", "s_nop 3", "v_accvgpr_read_b32 v20, a1", "s_endpgm"]
    size = [16, 4, 4, 4, 4, 8, 4]
    lines, address = [], 0
    for c, n in zip(code, size):
        lines.append(f"\t{c} // {address:012X}: 00000000")
        address += n
    bad, least = Function(lines).too_early()
    assert [(b[1], b[2], b[3]) for b in bad] == [("v_accvgpr_read_b32 v20, a1", 5, 12)] and least == -7
    straight = [l for l in lines if "cbranch" not in l]
    assert Function(straight).too_early() == ([], 0)
    assert needed(product + " blgp:4") == 8 and registers("v[2:3], a7") == {("v", 2), ("v", 3), ("a", 7)}
