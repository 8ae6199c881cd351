"""The scaled matrix instruction with one operand of 8 bits and one of 4: the compiler waits for its result as if both had 4, too short, so
the kernels write it in one statement with a wait of their own.  Used through the builtin, a copy that the compiler places ahead of a
separate wait would read registers that are not written yet, without an error."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(__file__), "..", "qwen3-tts-engine_amd", "csrc")


def _code(path):
    with open(path) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_every_scaled_product_is_in_one_statement_with_its_wait():
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        code = _code(path)
        assert "builtin_amdgcn_mfma_scale" not in code, path
        statements = re.findall(r"\basm\b[^;]*?\((.*?)\);", code, re.S)
        inside = [s for s in statements if "v_mfma_scale" in s]
        assert code.count("v_mfma_scale") == sum(s.count("v_mfma_scale") for s in inside), path
        for s in inside:
            text = re.split(r"\n\s*:", s)[0]                           # ahead of the operands
            lines = "".join(re.findall(r'"([^"]*)"', text)).replace("\\t", "").split("\\n")
            products = [i for i, x in enumerate(lines) if x.startswith("v_mfma_scale")]
            assert lines[-1] == "s_nop 15" and products == list(range(1, len(lines) - 1)) and lines[0] == "s_nop 1", (path, lines)
            # results apart from every operand: the second product is not to read what the first one has written
            outputs = re.findall(r'"(=[^"]*)"', s)
            assert len(outputs) == len(products) and set(outputs) == {"=&v"}, (path, outputs)
            found += 1
    assert found == 1
