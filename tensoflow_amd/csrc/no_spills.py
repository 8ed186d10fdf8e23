"""Reads what hipcc reports with -Rpass-analysis=kernel-resource-usage; fails for a kernel that spills vector registers, uses scratch memory or a dynamic stack.

The scan kernels keep a tile's rows in registers.  One that was held to fewer than it needs (a backward kernel of four 16-bit channels: 128, 63 of them
spilled) gave wrong states in one of its channels, and no mistake was found in its source: until one is, no kernel of theirs is built that way.
Spilled SCALAR registers (lanes of vector registers; the forward kernels have 75 to 106, the backward ones 102 to 181) are not refused."""
import re
import sys

LIMITS = {"VGPRs Spill": "0", "ScratchSize [bytes/lane]": "0", "Dynamic Stack": "False"}


def kernels(text):
    """{kernel: {what: value}}"""
    out, name = {}, None
    for what, value in re.findall(r"remark: .*?([A-Z][\w\[\]/ ]*): (\S+)", text):
        if what == "Function Name":
            name = value
            out[name] = {}
        elif name:
            out[name][what] = value
    return out


def main(path):
    text = open(path).read()
    for line in sorted({m for m in re.findall(r"^.*warning: .*$", text, re.M)}):
        print(line, file=sys.stderr)
    found = kernels(text)
    bad = [f"{name}: {what} {got.get(what, 'not reported')}" for name, got in found.items() for what, want in LIMITS.items() if got.get(what) != want]
    for line in bad:
        print(f"{path}: {line}", file=sys.stderr)
    if not found:
        print(f"{path}: no kernel reported", file=sys.stderr)
    return 1 if bad or not found else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1]))
