"""The copies from memory straight to LDS: what their instructions need around them."""
import os
import re


def statements(text):
    """The instruction strings of the inline assembly in a source, comments taken out."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\(((?:\s*\"(?:[^\"\\]|\\.)*\")+)", text):
        code = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
        yield [i.strip() for i in re.split(r"\\n|\\t|\n|;", code) if i.strip()]


def test_a_wait_state_between_m0_and_the_copy_that_reads_it():
    """The instruction set asks software for one wait state between a scalar write of M0 and a load to LDS.  The compiler puts
    it in for its own code and does not look into inline assembly, so every statement with such a load writes M0 itself, with
    one other instruction in between."""
    from prime_moe import build
    copies = 0
    for name in sorted(os.listdir(build.CSRC)):
        if not name.endswith((".h", ".hip")):
            continue
        for code in statements(open(os.path.join(build.CSRC, name)).read()):
            writes = [i for i, c in enumerate(code) if re.match(r"s_\w+\s+m0\s*,", c)]
            for at, c in enumerate(code):
                if not re.match(r"(global|buffer|scratch)_load_lds|.*\blds\s*$", c):
                    continue
                copies += 1
                before = [w for w in writes if w < at]
                assert before and at - before[-1] >= 2, (name, code)
    assert copies >= 7
