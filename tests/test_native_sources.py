"""The native sources: what they include, and where a copy of them compiles (CPU)."""
import pathlib
import re
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "comfyui-rdna35-attention_b200" / "csrc"
FILES = sorted(p for folder in (CSRC, ROOT / "include") for p in folder.iterdir() if p.suffix in (".cu", ".cuh", ".h"))


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_includes_are_relative_to_their_file(path):
    for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', path.read_text(), re.M):
        assert not pathlib.PurePath(name).is_absolute(), f"{path.name} includes {name}"
        assert (path.parent / name).is_file(), f"{path.name} includes {name}, which is not there"


def test_a_copy_elsewhere_reads_its_own_headers(tmp_path):
    import build_native

    try:
        nvcc = build_native._nvcc()
    except RuntimeError as reason:
        pytest.skip(str(reason))
    copy = tmp_path / "checkout"
    shutil.copytree(CSRC, copy / CSRC.relative_to(ROOT))
    shutil.copytree(ROOT / "include", copy / "include")
    lists = [(src.name, subprocess.Popen([nvcc, *build_native.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I",
                                          str(copy / "include"), "-M", str(copy / CSRC.relative_to(ROOT) / src.name)],
                                         stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True))
             for src in build_native.sources()]
    for name, proc in lists:
        out, err = proc.communicate()
        assert proc.returncode == 0, f"{name}: {err}"
        deps = [pathlib.Path(d).resolve() for d in out.replace("\\\n", " ").split(":", 1)[1].split()]
        foreign = [str(d) for d in deps if ROOT in d.parents]
        assert not foreign, f"{name} of the copy reads {foreign}"


# Instructions that copy to or wait for memory which ordinary loads and stores read and write: without the clobber the
# compiler may move those across them.
MEMORY = re.compile(r"\b(cp\.async|mbarrier\.|fence\.|bar\.sync|griddepcontrol\.)")


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_copies_and_waits_clobber_memory(path):
    for match in re.finditer(r"\basm\s+volatile\s*\((.*?)\)\s*;", path.read_text(), re.S):
        if MEMORY.search(match[1]):
            assert '"memory"' in match[1], f"{path.name}: {match[0]}"
