"""Scan of the experts' product kernels (gfx950 assembly of expert_gemm.hip) for the buffer descriptors of their
panel loads: wherever a `buffer_load ... lds` can be reached from, the four scalar registers of its
descriptor have been written, the last one with the type word 0x20000. The compiler once left a descriptor
unwritten on one edge (no tile is left) though the source sets it on all: such a load reads anywhere.

A register counts as holding the word if it does on every path (moves and registers kept in a vector
register's lanes are followed); a block starts from what holds on all of its edges."""
import re

WORD = 0x20000


def _regs(text):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", text)
    if m:
        return list(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.fullmatch(r"s(\d+)", text)
    return [int(m.group(1))] if m else []


def _blocks(lines):
    """[(labels, instructions)] in order."""
    out = [([], [])]
    for raw in lines:
        text = raw.split(";")[0].strip()
        if not text:
            continue
        if text.endswith(":"):
            if out[-1][1]:
                out.append(([], []))
            out[-1][0].append(text[:-1])
        elif not text.startswith("."):
            out[-1][1].append(text)
            if re.match(r"s_c?branch|s_endpgm|s_setpc", text):
                out.append(([], []))
    return out


def _step(state, text):
    """What holds after an instruction: registers, and (vector register, lane) pairs, with the word in them."""
    op, _, rest = text.partition(" ")
    ops = [o.strip() for o in rest.split(",")]
    if op == "v_writelane_b32":
        slot = (ops[0], ops[2])
        return state | {slot} if set(_regs(ops[1])) & state else state - {slot}
    if op == "v_readlane_b32":
        r = set(_regs(ops[0]))
        return state | r if (ops[1], ops[2]) in state else state - r
    if op in ("s_mov_b32", "s_mov_b64") and len(ops) == 2:
        to, source = _regs(ops[0]), _regs(ops[1])
        if source:
            held = [r in state for r in source]
        else:
            try:
                held = [int(ops[1], 0) == WORD] + [False] * (len(to) - 1)
            except ValueError:
                held = [False] * len(to)
        return (state - set(to)) | {r for r, h in zip(to, held) if h}
    if op.startswith(("buffer_", "global_", "scratch_", "ds_", "s_cmp", "s_waitcnt", "s_barrier", "s_nop", "s_cbranch",
                      "s_branch", "s_endpgm", "s_bitcmp")):
        return state
    # a result is the first operand, a carry or a mask the second
    gone = set(_regs(ops[0])) if ops else set()
    if op.startswith("v_") and len(ops) > 1 and ("_co_" in op or op.startswith("v_div_scale")):
        gone |= set(_regs(ops[1]))
    return state - gone


def scan(lines):
    """The loads, with the block's number, whose descriptor's last word is not set on some path."""
    blocks = _blocks(lines)
    at = {label: i for i, (labels, _) in enumerate(blocks) for label in labels}
    edges = []
    for i, (_, code) in enumerate(blocks):
        last = code[-1] if code else ""
        to = [at[m.group(1)] for m in [re.match(r"s_c?branch\S*\s+(\S+)", last)] if m and m.group(1) in at]
        if not re.match(r"s_branch|s_endpgm|s_setpc", last) and i + 1 < len(blocks):
            to.append(i + 1)
        edges.append(to)
    entry = [None] * len(blocks)
    entry[0] = frozenset()
    todo = [0]
    while todo:
        i = todo.pop()
        state = set(entry[i])
        for text in blocks[i][1]:
            state = _step(state, text)
        for j in edges[i]:
            new = frozenset(state) if entry[j] is None else entry[j] & frozenset(state)
            if new != entry[j]:
                entry[j] = new
                todo.append(j)
    found = []
    for i, (_, code) in enumerate(blocks):
        if entry[i] is None:
            continue
        state = set(entry[i])
        for text in code:
            m = re.match(r"buffer_load\S* \S+ s\[(\d+):(\d+)\].*\blds$", text)
            if m and int(m.group(2)) not in state:
                found.append((i, text))
            state = _step(state, text)
    return found
