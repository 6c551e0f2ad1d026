"""How the library is compiled."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genre-shapehd_amd", "csrc")


def test_no_source_is_compiled_with_packed_fp32():
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, timeout=120, check=True).stdout.splitlines()
    compiled = [line.split() for line in lines if ".hip -o " in line and " -c " in line]
    assert {words[words.index("-c") + 1] for words in compiled} == {f for f in os.listdir(CSRC) if f.endswith(".hip")}
    for words in compiled:
        at = words.index("-packed-fp32-ops")
        assert words[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"] and "-ffp-contract=off" in words


def test_variants_of_the_library_hold_every_object():
    """tools/build_variants.sh links one recompiled source with the other objects of the library"""
    with open(os.path.join(CSRC, "..", "..", "tools", "build_variants.sh")) as f:
        listed = next(line for line in f if line.startswith("for o in "))
    assert {o + ".hip" for o in listed[len("for o in "):listed.index(";")].split()} == {f for f in os.listdir(CSRC) if f.endswith(".hip")}


def test_build_compiles_whatever_is_built_already(genre, monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(subprocess, "check_call", calls.append)
    monkeypatch.setattr(subprocess, "call", lambda *args, **kwargs: 3)
    entry.build()
    assert CSRC in calls[0] and all(words[0] == "make" and "-B" in words for words in calls)
