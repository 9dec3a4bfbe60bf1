"""The codes that kernels leave in the status word: each belongs to one source file and has a text of its own that names it."""
import ast
import re
from pathlib import Path

from spissa_b200.csrc import lib

CSRC = Path(lib.__file__).parent
NAMES = {"tc_gemm": "", "flash_tc": "attention:", "tc_stream": "tc_stream:", "tc_mid": "tc_mid:", "tc_f32": "tc_f32:", "rglru_kernels": "rglru:",
         "mlstm_kernels": "mlstm:", "kv4_attention": "kv4_attention:", "q4_tc": "q4_tc:", "decode_layers": "decode layers:"}


def waits():
    """{source: codes of its bounded waits}."""
    found = {}
    for path in sorted(CSRC.glob("*.cu")):
        codes = {int(c) for c in re.findall(r"(?:wait\w*|wait_for)\([^;{}]*?status,\s*(\d{3})\b", path.read_text())}
        if codes:
            found[path.stem] = codes
    return found


def test_a_code_belongs_to_one_kernel_and_its_text_names_it():
    found = waits()
    assert {"q4_tc", "kv4_attention", "rglru_kernels", "mlstm_kernels", "tc_f32", "tc_gemm", "flash_tc"} <= set(found)
    owner = {}
    for source, codes in found.items():
        for code in codes:
            assert owner.setdefault(code, source) == source, f"code {code} is recorded by {owner[code]} and by {source}"
            assert code in lib.STATUS_TEXT and lib.STATUS_TEXT[code].startswith(NAMES[source]), (source, code, lib.STATUS_TEXT.get(code))
    assert all(len(codes) > 1 for codes in found.values())


def test_no_text_is_given_twice():
    tree = ast.parse((CSRC / "lib.py").read_text())
    table = next(n.value for n in tree.body if isinstance(n, ast.Assign) and getattr(n.targets[0], "id", "") == "STATUS_TEXT")
    keys = [k.value for k in table.keys]
    assert len(keys) == len(set(keys)), sorted(k for k in keys if keys.count(k) > 1)
