"""The in-tree build: when a target is built again.  No compiler runs here."""
import os
import subprocess

import pytest

from vits_amd import build as b


def remarks(*kernels):
    """What the compiler says of its kernels' registers (-Rpass-analysis=kernel-resource-usage)."""
    lines = []
    for name, change in kernels:
        says = {"TotalSGPRs": 90, "VGPRs": 256, "AGPRs": 0, "ScratchSize [bytes/lane]": 0, "Dynamic Stack": "False", "Occupancy [waves/SIMD]": 2,
                "SGPRs Spill": 72, "VGPRs Spill": 0, "LDS Size [bytes/block]": 16852, **change}
        lines += [f"/a/b.hip:52:1: remark: {x} [-Rpass-analysis=kernel-resource-usage]\n   52 | __global__ void f() {{\n      | ^" for x in
                  (f"Function Name: {name}", *(f"    {k}: {v}" for k, v in says.items()))]
    return "\n".join(lines) + "\n"


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The build in an empty library folder, with compilers that only write down what they were asked for."""
    ran, used = [], [("some_kernel", {})]

    def compiler(cmd, check=True, **kw):
        ran.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", remarks(*used))
    for name in ("LIBDIR", "LIB", "BINDING"):
        monkeypatch.setattr(b, name, str(tmp_path / os.path.basename(getattr(b, name))) if name != "LIBDIR" else str(tmp_path))
    monkeypatch.setattr(b.subprocess, "run", compiler)

    def built():
        ran.clear()
        b.build(verbose=False)
        return sorted(os.path.basename(cmd[cmd.index("-o") + 1]) for cmd in ran)
    built.used = used
    return built


EVERYTHING = sorted([s.replace(".hip", ".o") for s in b.SOURCES] + ["_vits_ops.so", "libvits_amd.so"])


def test_a_second_build_has_nothing_to_do(tree):
    assert tree() == EVERYTHING
    assert tree() == []


def test_other_flags_build_again(tree, monkeypatch):
    tree()
    monkeypatch.setattr(b, "FLAGS", b.FLAGS + ["-DOTHER"])
    assert tree() == sorted(x for x in EVERYTHING if x != "_vits_ops.so")
    assert tree() == []
    monkeypatch.setattr(b, "SOURCE_FLAGS", {"kernels_gl16.hip": ["-DONE"], **b.SOURCE_FLAGS})
    assert tree() == ["kernels_gl16.o", "libvits_amd.so"]
    monkeypatch.setattr(b, "CXX", "another-compiler")
    assert tree() == ["_vits_ops.so"]
    monkeypatch.setattr(b, "HIPCC", "another-hipcc")
    assert tree() == sorted(x for x in EVERYTHING if x != "_vits_ops.so")


def test_objects_of_an_unknown_command_are_built_again(tree):
    """A folder that holds objects of an earlier build, which nothing says the flags of."""
    for name in EVERYTHING:
        with open(os.path.join(b.LIBDIR, name), "w") as f:
            f.write("from before")
    assert tree() == EVERYTHING


def test_the_binding_follows_the_header(tree):
    """The binding's calls are declared by include/vits_amd.h alone: it includes it, and is built again with it."""
    tree()
    header = os.path.join(os.path.dirname(b.HERE), "include", "vits_amd.h")
    with open(os.path.join(b.CSRC, "ops_binding.cpp")) as f:
        source = f.read()
    assert '#include "../../include/vits_amd.h"' in source and "decltype(&vits_op_paged_attention)" in source
    later = os.path.getmtime(header) + 10
    for name in EVERYTHING:
        os.utime(os.path.join(b.LIBDIR, name), (later, later))
    real = os.path.getmtime
    b_getmtime = lambda path: later + 1 if path == header else real(path)      # noqa: E731
    with pytest.MonkeyPatch.context() as m:
        m.setattr(b.os.path, "getmtime", b_getmtime)
        assert set(tree()) >= {"_vits_ops.so", "model.o", "kernels_paged.o", "libvits_amd.so"}


def test_the_build_check_compiles_everything(tree, monkeypatch):
    """__graft_entry__.build() says whether the tree builds, so it compiles whatever is there already."""
    import __graft_entry__ as entry
    tree()
    asked = []
    monkeypatch.setattr(b, "build", lambda **kw: asked.append(kw) or os.path.join(b.LIBDIR, "libvits_amd.so"))
    entry.build()
    assert asked == [dict(force=True)]


@pytest.mark.parametrize("change,word", [({"AGPRs": 2}, "AGPRs"), ({"VGPRs": 257}, "VGPRs"), ({"ScratchSize [bytes/lane]": 16}, "ScratchSize"),
                                         ({"VGPRs Spill": 3}, "VGPRs Spill")])
def test_a_build_of_too_many_registers_is_none(tree, change, word):
    """The paged attention has to stay within 256 vector registers, without accumulator registers and scratch."""
    tree.used[:] = [("one", {}), ("another", change)]
    with pytest.raises(RuntimeError, match=f"another.*{word}"):
        tree()
    tree.used[:] = [("one", {}), ("another", {})]
    assert {"kernels_paged.o", "libvits_amd.so"} <= set(tree())                     # what was refused is not taken for built
    assert tree() == []


def test_a_build_that_says_nothing_of_its_registers_is_none(tree):
    tree.used.clear()
    with pytest.raises(RuntimeError, match="registers"):
        tree()


def test_other_messages_of_the_compiler_are_passed_on():
    odd, end = "x.hip:3:4: warning: odd\n    3 | int x;\n      | ^\n", "1 warning generated.\n"
    assert b._check_registers("x.hip", odd + remarks(("one", {})) + end) == odd + end
