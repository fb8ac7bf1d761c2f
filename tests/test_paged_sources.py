"""What the compiler has to know of the inline assembly in hearth_amd/csrc, read from the sources and
from the assembly that it makes of them."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

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


def _unwritten(asm):
    """(statements with LDS loads, those that do not have exactly one write of m0 between the one
    before and themselves)"""
    writes = total = bad = 0
    inside = loads = False
    for line in asm.splitlines():
        t = line.strip()
        if t.startswith(";;#ASMSTART"):
            inside, loads = True, False
        elif t.startswith(";;#ASMEND"):
            inside = False
            if loads:
                total, bad, writes = total + 1, bad + (writes != 1), 0
        elif inside:
            loads = loads or "_lds_" in t
        elif re.match(r"s_\w+\s+m0\b", t):
            writes += 1
    return total, bad


@pytest.mark.parametrize("name", ["k_paged_many.hip", "k_paged_latent.hip"])
def test_m0_is_written_before_each_statement(name, tmp_path):
    """As the compiler places them: nothing comes between a statement's write of m0 and the statement."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc is not available")
    out = tmp_path / "k.s"
    flags = [f for f in build.COMMON if f != "-fPIC"]
    r = subprocess.run([hipcc, "-x", "hip", *flags, "--cuda-device-only", "-S", str(build.CSRC / name), "-o", str(out)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    total, bad = _unwritten(out.read_text())
    assert total >= 8 and bad == 0, (total, bad)


def test_the_check_sees_a_write_between():
    block = ";;#ASMSTART\ns_nop 0\nglobal_load_lds_dwordx4 v1, s[0:1]\n;;#ASMEND\n"
    assert _unwritten("s_mov_b32 m0, s1\n" + block) == (1, 0)
    assert _unwritten("s_mov_b32 m0, s1\ns_mov_b32 m0, s2\n" + block) == (1, 1)
    assert _unwritten("s_mov_b32 m0, s1\n" + block + block) == (2, 1)


def test_scales_are_read_at_any_address():
    """A cache's scale bytes may lie at any address: wider reads of them go through types that say so."""
    text = COMMENT.sub(" ", (build.CSRC / "k_paged_attn.hip").read_text())
    reads = re.findall(r"\(const (\w+) \*\)\(?q\b", text)
    assert len(reads) >= 4 and all(t.endswith("_any") for t in reads), reads
    header = (build.CSRC / "hx_paged.h").read_text()
    for t in set(reads):
        assert re.search(rf"typedef [\w ]+ {t} __attribute__\(\(aligned\(1\)\)\);", header), t
