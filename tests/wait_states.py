"""Wait states that gfx950 leaves to software, looked for in the compiler's assembly of the kernels.

The compiler pads its own instructions, but not what stands in inline assembly.  Looked for are

* a vector memory instruction that reads an SGPR which a vector instruction wrote: 5 wait states;
* a load into LDS after a scalar instruction wrote M0: 1;
* a vector instruction of inline assembly that reads or writes what a matrix instruction writes: the passes of that and 4; that
  writes the addend of one: its passes.  (A pass is 4 cycles: 32 x 32 x 16 products at 1024 operations a cycle and SIMD take 8, 16 x 16 x
  32 take 4, and half as deep ones no longer; any other shape is taken for the longest, 16.)

An instruction is one wait state, ``s_nop n`` is n + 1.  Each kernel is followed along its branches.
"""
import re
from collections import deque

_REG = re.compile(r"(?<![\w.])([sva])(?:(\d+)|\[(\d+):(\d+)\])(?![\w\[])")
_SALU_NO_SDST = ("s_nop", "s_wait", "s_barrier", "s_branch", "s_cbranch", "s_cmp", "s_bitcmp", "s_endpgm", "s_setprio", "s_sleep", "s_setreg",
                 "s_sendmsg", "s_store", "s_dcache", "s_icache", "s_trap", "s_sethalt")
_VMEM = ("buffer_", "global_", "flat_", "scratch_", "tbuffer_")
_FAR = 64


def _regs(text):
    out = set()
    for kind, one, lo, hi in _REG.findall(text):
        out.update((kind, i) for i in (range(int(lo), int(hi) + 1) if lo else (int(one),)))
    for name in ("vcc", "m0", "exec"):
        if re.search(rf"\b{name}\b", text):
            out.update({("s", "vcc_lo"), ("s", "vcc_hi")} if name == "vcc" else {("s", name)})
    for name in ("vcc_lo", "vcc_hi"):
        if re.search(rf"\b{name}\b", text):
            out.add(("s", name))
    return out


class Instruction:
    __slots__ = ("name", "text", "line", "inline", "states", "dst", "src", "lds")

    def __init__(self, text, line, inline):
        self.text, self.line, self.inline = text, line, inline
        self.name, _, rest = text.partition(" ")
        self.name = self.name.strip()
        ops, depth, cur = [], 0, ""
        for ch in rest:
            depth += (ch == "[") - (ch == "]")
            if ch == "," and depth == 0:
                ops.append(cur)
                cur = ""
            else:
                cur += ch
        ops.append(cur)
        self.states = int(rest.strip(), 0) + 1 if self.name == "s_nop" else 1
        self.lds = self.name.startswith(_VMEM) and re.search(r"\blds\b", rest) is not None
        n = 0
        if self.valu:
            n = 1
            # a second result: the carry, or div_scale's flag
            if re.match(r"v_(add|sub|subrev|addc|subb|subbrev)_co_|v_div_scale|v_mad_[ui]64", self.name):
                n = 2
            elif re.match(r"v_swap|v_permlane(16|32)_swap", self.name):
                n = 2
            elif self.name.startswith("v_nop"):
                n = 0
        elif self.name.startswith("s_") and not self.name.startswith(_SALU_NO_SDST):
            n = 1
        self.dst = set().union(*(_regs(o) for o in ops[:n])) if n else set()
        self.src = set().union(*(_regs(o) for o in ops[n:])) if ops[n:] else set()
        if n == 2 and "swap" in self.name:
            self.src |= self.dst
        if self.name.startswith("v_cmp") and not self.name.startswith("v_cmpx") and "_e32" in self.name:
            self.dst |= {("s", "vcc_lo"), ("s", "vcc_hi")}

    @property
    def valu(self):
        return self.name.startswith("v_")

    @property
    def vmem(self):
        return self.name.startswith(_VMEM)

    @property
    def mfma(self):
        return self.name.startswith(("v_mfma", "v_smfmac"))

    def mfma_passes(self):
        m = re.match(r"v_mfma_f32_(32x32x(?:8|16)|16x16x(?:16|32))_?b?f16", self.name)
        return 16 if not m else 8 if m.group(1).startswith("32") else 4

    def addend(self):
        return _regs(self.text.split(",", 1)[1].rsplit("]", 1)[0].rsplit(",", 1)[-1] + "]") if self.mfma else set()


def _functions(assembly):
    """(name, blocks: {label: ([instructions], [labels that follow])}, first label) of each function."""
    name, blocks, label, first, inline, open_ = None, {}, None, None, False, True
    for number, raw in enumerate(assembly.splitlines(), 1):
        line = raw.split("//")[0]
        if ";;#ASMSTART" in line or ";;#ASMEND" in line:
            inline = "START" in line
            continue
        line = line.split(";")[0].rstrip()
        if not line.strip():
            continue
        m = re.match(r"^([.\w$]+):", line)
        if m:
            at = m.group(1)
            if at.startswith(".Lfunc_end"):
                if name:
                    yield name, blocks, first
                name, blocks, label = None, {}, None
            elif at.startswith(".L") and name:
                if label is not None and open_:
                    blocks[label][1].append(at)
                blocks[at], label, open_ = ([], []), at, True
            elif not at.startswith(".L"):
                name, blocks, label, first, open_ = at, {at: ([], [])}, at, at, True
            continue
        text = line.strip()
        if name is None or text.startswith("."):
            continue
        if not open_:  # behind a branch: a block of its own
            label = f"{label}+{number}"
            blocks[label], open_ = ([], []), True
            if blocks[last][0][-1].name.startswith("s_cbranch"):
                blocks[last][1].append(label)
        i = Instruction(text, number, inline)
        blocks[label][0].append(i)
        if i.name in ("s_branch", "s_endpgm", "s_setpc_b64") or i.name.startswith("s_cbranch"):
            if "branch" in i.name:
                blocks[label][1].append(text.split()[-1])
            last, open_ = label, False


def _walk(instructions, state, found):
    """``state``: {(rule, register): wait states since}; returns it after the instructions."""
    def put(key, least):
        old = state.get(key)
        state[key] = least if old is None else min(old, least)

    for i in instructions:
        if i.vmem:
            regs = i.src | i.dst
            for r in regs:
                age = state.get(("valu", r))
                if age is not None and age < 5:
                    found[(i.line, "sgpr")] = (i.line, i.text, f"{r[0]}{r[1]} written by a vector instruction {age} wait states before, 5 needed")
            age = state.get(("salu", ("s", "m0")))
            if i.lds and age is not None and age < 1:
                found[(i.line, "m0")] = (i.line, i.text, "m0 written immediately before, 1 wait state needed")
        if i.inline and i.valu and not i.mfma:
            for r in i.src | i.dst:
                age = state.get(("mfma", r))
                if age is not None and age < 0:
                    found[(i.line, "mfma")] = (i.line, i.text, f"{r[0]}{r[1]} of a matrix instruction {-age} wait states too early")
            for r in i.dst:
                age = state.get(("addend", r))
                if age is not None and age < 0:
                    found[(i.line, "addend")] = (i.line, i.text, f"{r[0]}{r[1]} read by a matrix instruction, {-age} wait states too early")
        for key in list(state):
            if state[key] + i.states >= _FAR:
                del state[key]
            else:
                state[key] += i.states
        for r in i.dst:
            if r[0] == "s":
                state.pop(("valu", r), None)
                if i.valu:
                    state["valu", r] = 0
                elif r == ("s", "m0"):
                    state["salu", r] = 0
        if i.mfma:
            for r in i.dst:
                state["mfma", r] = -(i.mfma_passes() + 4)
            for r in i.addend():
                put(("addend", r), -i.mfma_passes())
        elif i.valu:
            # (what the compiler's own instruction writes it has waited for)
            for r in i.dst:
                if not i.inline:
                    state.pop(("mfma", r), None)
    return state


def missing(assembly):
    """[(line, instruction, what is missing)] of the assembly of a source file."""
    found = {}
    for _, blocks, first in _functions(assembly):
        at = {first: {}}
        queue = deque([first])
        while queue:
            label = queue.popleft()
            state = _walk(blocks[label][0], dict(at[label]), found)
            for to in blocks[label][1]:
                if to not in blocks:
                    continue
                old, new = at.get(to), dict(state)
                if old is not None:
                    new = dict(old)
                    for k, v in state.items():
                        new[k] = min(new.get(k, v), v)
                    if new == old:
                        continue
                at[to] = new
                queue.append(to)
    return sorted(found.values())
