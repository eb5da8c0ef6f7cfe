"""What the sources, documents, profiles and tools of the tree may hold (CPU)."""
import os
import re

from conftest import ROOT

PARTS = ("nextpolish_amd", "include", "tests", "tools", "oracle", "docs", "profiles",
         "DESIGN.md", "INTEGRATION.md", "README.md", "bench.py", "__graft_entry__.py", "pytest.ini")
KINDS = (".py", ".sh", ".c", ".cpp", ".h", ".hip", ".md", ".txt", ".ini", "Makefile")


def texts():
    """(path relative to the root, text) of every source, script, document and profile; built files, fixtures and this file are left out."""
    for part in PARTS:
        top = os.path.join(ROOT, part)
        for d, dirs, names in os.walk(top) if os.path.isdir(top) else [(ROOT, [], [part])]:
            dirs[:] = [x for x in dirs if x not in ("__pycache__", "build", "lib", "bin", "_ref", "golden")]
            for n in sorted(names):
                p = os.path.join(d, n)
                if n.endswith(KINDS) and p != os.path.abspath(__file__):
                    with open(p, errors="replace") as f:
                        yield os.path.relpath(p, ROOT), f.read()


def test_no_text_reads_offsets_of_an_installed_library():
    # An offset into a library that was not built here is only ever part of an unannotated back trace, "lib.so.N(+0x...)[0x...]": a text that
    # gives one a meaning rests on the library's code.
    trace = re.compile(r"\S+\.so\.\d+\(\S*\+0x[0-9a-f]+\)\[0x[0-9a-f]+\]")
    offset = re.compile(r"\+0x[0-9a-f]{4,}")
    bad = []
    for path, text in texts():
        for k, line in enumerate(text.splitlines(), 1):
            rest = re.sub(r"\S+/nextpolish_amd/lib/\S+", "", trace.sub("", line))      # (offsets into the project's own libraries are its own)
            if offset.search(rest):
                bad.append("%s:%d" % (path, k))
    assert not bad, bad


def test_every_tool_that_a_text_names_is_there():
    # (a document may name a tool with or without its folder; "name*" stands for several)
    named = re.compile(r"\b(?:tests/)?tools/([A-Za-z0-9_]+(?:/[A-Za-z0-9_]+)?\.(?:sh|py|hip|cpp))")
    have = {os.path.relpath(os.path.join(d, n), os.path.join(ROOT, top))
            for top in ("tests/tools", "tools") for d, _, names in os.walk(os.path.join(ROOT, top)) for n in names}
    bad = sorted({(path, m) for path, text in texts() for m in named.findall(text) if m not in have})
    assert not bad, bad


def test_nothing_repeats_the_test_runner_or_a_test_until_it_fails():
    bad = []
    for path, text in texts():
        if path.endswith(".sh") and re.search(r"^\s*for \w+ in \$\(seq", text, re.M) and "pytest" in text:
            bad.append(path)
        if path.endswith(".py") and re.search(r"parametrize\(.*os\.environ", text):
            bad.append(path)
    assert not bad, bad


def test_the_tools_hold_no_gpu_program_and_nothing_registers_memory_that_exists():
    bad = []
    for path, text in texts():
        if path.startswith(("tests/tools", "tools")) and (path.endswith(".hip") or re.search(r"^[^#\n]*\bhipcc\b", text, re.M)):
            bad.append(path)      # (GPU code is built by nextpolish_amd/csrc/Makefile only)
        if path.endswith((".hip", ".cpp", ".h", ".c")) and re.search(r"\bhipHostRegister\s*\(", text):
            bad.append(path)
    assert not bad, bad


def test_device_memory_comes_from_plain_allocations():
    # (no buffer is placed against an unmapped page: an access out of range is looked for in the host models, not by a fault)
    bad = [path for path, text in texts() if path.startswith("nextpolish_amd") and re.search(r"\bhipMem(AddressReserve|Create|Map|SetAccess)\b", text)]
    assert not bad, bad


def test_the_user_document_names_the_switches_that_are_read_and_no_others():
    src = "".join(text for path, text in texts() if path.startswith("nextpolish_amd") or path in ("bench.py",))
    read = re.compile(r'(?:getenv|env_\w+|environ\w*(?:\.get)?)[(\[]\s*"(NP[12]?_[A-Z][A-Z0-9_]*)"')
    with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
        named = set(re.findall(r"\bNP[12]?_[A-Z][A-Z0-9_]*", f.read()))
    libs = set(read.findall("".join(text for path, text in texts() if path.startswith("nextpolish_amd"))))
    assert len(named) > 20 and len(libs) > 20
    assert not named - set(read.findall(src)), sorted(named - set(read.findall(src)))
    assert not libs - named, sorted(libs - named)


def test_no_switch_makes_a_result_wrong():
    # a build that leaves work out to time the rest is no part of the tree
    said = re.compile(r"results are wrong when|output is wrong|wrong output|experiments with wrong results|parts of the work left out")
    bad = ["%s:%d" % (path, k) for path, text in texts() if path.startswith(("nextpolish_amd", "include", "bench.py"))
           for k, line in enumerate(text.splitlines(), 1) if said.search(line)]
    assert not bad, bad


def test_no_device_source_ends_the_process():
    # (the drop-in symbols exit where the reference's do, on the host; code that launches kernels could leave them running behind it)
    bad = []
    for path, text in texts():
        if path.startswith("nextpolish_amd/csrc") and path.endswith(".hip"):
            if re.search(r"\b(_exit|_Exit|quick_exit|exit|abort)\s*\(", re.sub(r"//[^\n]*", "", text)):
                bad.append(path)
    assert not bad, bad


def test_hip_sources_are_compiled_without_packed_fp32():
    with open(os.path.join(ROOT, "nextpolish_amd", "csrc", "Makefile")) as f:
        text = f.read()
    flags = re.search(r"^HIPFLAGS *:=(.*)$", text, re.M).group(1)
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in flags
    assert re.search(r"\$\(HIPCC\) \$\(HIPFLAGS\) -c", text) and len(re.findall(r"\$\(HIPCC\)[^\n]* -c ", text)) == 1
    bad = [path for path, body in texts() if path.startswith("nextpolish_amd") and re.search(r"v_pk_(add|mul|fma)_f32", body)]
    assert not bad, bad


def test_the_sources_stand_on_their_own():
    # what a comment says can be read without the documents beside the tree
    away = re.compile(r"\b[A-Z]{5,}\.md\b|§|\b[A-Z]{6,} r\d\b|\b[Rr]ound[s-]? ?[3-9]\b")
    bad = ["%s:%d" % (path, k) for path, text in texts() if path.startswith(("nextpolish_amd", "include", "oracle", "bench.py", "pytest.ini"))
           for k, line in enumerate(text.splitlines(), 1) if away.search(re.sub(r"SAMv1 §[\d., §]+", "", line))]
    assert not bad, bad
