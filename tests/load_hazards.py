"""Hazard scan of the experts' product kernels (gfx950 assembly of expert_gemm.hip), whose panel loads
are inline asm that the compiler's hazard recognizer does not look into: a scalar register that a vector
instruction wrote (v_readfirstlane, v_cmp) takes 5 wait states before a vector memory instruction may
read it. Counted back from each load over the straight line before it and, at a label, from every branch
to it and from what falls through."""
import re

WAIT = 5


def kernels(path):
    """(name, lines) of every function of an assembly file, to its end: a kernel may end in several places."""
    out, cur = [], None
    for line in open(path):
        m = re.match(r"^([A-Za-z_][\w.$]*):", line)
        if m:
            cur = []
            out.append((m.group(1), cur))
        elif line.startswith(".Lfunc_end"):
            cur = None
        elif cur is not None:
            cur.append(line)
    return out


def scalars(text):
    out = set()
    for lo, hi, one in re.findall(r"\bs(?:\[(\d+):(\d+)\]|(\d+)\b)", text):
        out.update([int(one)] if one else range(int(lo), int(hi) + 1))
    return out


def _code(lines):
    out = []
    for raw in lines:
        text = raw.split(";")[0].strip()
        if text.endswith(":"):
            out.append(("label", text[:-1]))
        elif text and not text.startswith("."):
            out.append(("ins", text))
    return out


def scan(lines):
    code = _code(lines)
    jumps = {}
    for at, (kind, text) in enumerate(code):
        m = re.match(r"s_(?:c)?branch\S*\s+(\S+)", text) if kind == "ins" else None
        if m:
            jumps.setdefault(m.group(1), []).append(at)
    found = set()

    def back(at, left, used, load, seen):
        """The instructions before place `at`, as long as `left` wait states are wanted."""
        while left > 0 and at > 0:
            at -= 1
            kind, text = code[at]
            if kind == "label":
                if (at, left) in seen:
                    return
                seen.add((at, left))
                for j in jumps.get(text, ()):
                    back(j, left - 1, used, load, seen)
                continue
            if re.match(r"s_branch|s_endpgm|s_setpc", text) and code[at + 1][0] == "label":
                return  # nothing falls through
            if text.startswith("v_") and scalars(text.split(",")[0]) & used:
                found.add((text, load))
                return
            m = re.match(r"s_nop\s+(\d+)", text)
            left -= int(m.group(1)) + 1 if m else 1

    for at, (kind, text) in enumerate(code):
        if kind == "ins" and re.match(r"(buffer|global|scratch|flat)_", text):
            back(at, WAIT, scalars(text), text, set())
    return sorted(found)
