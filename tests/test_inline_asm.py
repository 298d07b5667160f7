"""Inline assembly of the kernels: what the compiler does for instructions that it knows and cannot do for these."""
import glob
import os
import re

from lastengine_amd import build

STORE = re.compile(r"(?:global|flat|buffer)_store_(?:dwordx[34]|b96|b128)")
TEXT = r'"((?:[^"\\]|\\.)*)"'  # a string literal


def blocks():
    """Each block's file and text, an element of which may be cut into several literals."""
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*"))):
        if path.endswith((".hip", ".h", ".cpp")):
            with open(path, encoding="utf-8") as f:
                for m in re.finditer(r"\basm(?:\s+volatile)?\s*\(\s*((?:%s\s*)+)" % TEXT, f.read()):
                    yield os.path.basename(path), "".join(re.findall(TEXT, m.group(1)))


def bare_stores(text):
    """Stores of more than 8 bytes without two wait states behind them in their block: until then their data registers may not be written,
    which the compiler keeps to for its own stores only."""
    lines = [i.strip() for i in re.split(r"\\n|\\t|;", text) if i.strip()]
    for i, line in enumerate(lines):
        if STORE.match(line):
            nop = re.match(r"s_nop (\d+)", lines[i + 1]) if i + 1 < len(lines) else None
            if not nop or int(nop.group(1)) < 1:
                yield line


def test_wide_stores_keep_their_wait_states():
    found = list(blocks())
    assert any(STORE.search(text) for _, text in found) and any("s_waitcnt" in text for _, text in found)  # they are read at all
    assert [(name, line) for name, text in found for line in bare_stores(text)] == []


def test_the_check_itself():
    assert list(bare_stores(r"global_store_dwordx4 %0, %1, off")) and list(bare_stores(r"global_store_dwordx4 %0, %1, off\n\ts_nop 0"))
    assert not list(bare_stores(r"global_store_dwordx4 %0, %1, off\n\ts_nop 1")) and not list(bare_stores(r"global_store_dwordx2 %0, %1, off"))
