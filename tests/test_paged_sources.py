"""What the compiler has to know of the inline assembly in hearth_amd/csrc, read from the sources."""
from __future__ import annotations

import re

import pytest

from hearth_amd import build

COMMENT = re.compile(r"/\*.*?\*/|//[^\n]*", re.S)


def _asms():
    """(file, statement) of every asm statement"""
    for src in sorted(p for p in build.CSRC.iterdir() if p.suffix in (".h", ".hip", ".cpp")):
        text = COMMENT.sub(" ", src.read_text())
        for m in re.finditer(r"\basm\b[^;]*?\(", text):
            depth, i = 1, m.end()
            while depth:
                if text[i] == '"':
                    i = re.compile(r'"(?:\\.|[^"\\])*"').match(text, i).end()
                    continue
                depth += {"(": 1, ")": -1}.get(text[i], 0)
                i += 1
            yield src.name, text[m.start():i]


ASMS = list(_asms())


def _template(stmt):
    """the instructions: the string literals before the first colon outside of one"""
    out = []
    for m in re.finditer(r'"((?:\\.|[^"\\])*)"|(:)', stmt):
        if m.group(2):
            break
        out.append(m.group(1))
    return "".join(out).replace("\\n", "\n").replace("\\t", "\t")


def _m0(stmt):
    """whether the statement leaves m0 as the compiler knows it"""
    lines = [ln.strip() for ln in _template(stmt).splitlines()]
    if any(re.match(r"s_\w+\s+m0\b", ln) for ln in lines):
        return False
    return not any("_lds_" in ln for ln in lines) or '"{m0}"' in stmt


@pytest.mark.parametrize("file,stmt", ASMS, ids=[f"{f}-{i}" for i, (f, _) in enumerate(ASMS)])
def test_m0_is_the_compilers(file, stmt):
    """m0, which LDS loads take their address from, is no register that a clobber list can name: an
    asm statement that writes it does so behind the compiler's back. It is taken as an input."""
    assert _m0(stmt), (file, stmt)


def test_the_check_sees_them():
    assert sum("_lds_" in _template(s) for f, s in ASMS if f == "hx_paged.h") == 3
    assert not _m0('asm volatile("s_mov_b32 m0, %0\\n\\tglobal_load_lds_dwordx4 %1, %2" ::"s"(a), "v"(o), "s"(b) : "memory")')
    assert not _m0('asm volatile("global_load_lds_dwordx4 %1, %2" ::"s"(a), "v"(o), "s"(b) : "memory")')


def test_scales_are_read_at_any_address():
    """A cache's scale bytes may lie at any address: wider reads of them go through types that say so."""
    text = COMMENT.sub(" ", (build.CSRC / "k_paged_attn.hip").read_text())
    reads = re.findall(r"\(const (\w+) \*\)\(?q\b", text)
    assert len(reads) >= 4 and all(t.endswith("_any") for t in reads), reads
    header = (build.CSRC / "hx_paged.h").read_text()
    for t in set(reads):
        assert re.search(rf"typedef [\w ]+ {t} __attribute__\(\(aligned\(1\)\)\);", header), t
