"""What the build is to have made of the device sources (no GPU needed)."""
import os
import re
import subprocess

import pytest

import __graft_entry__ as ge

LLVM = "/opt/rocm/lib/llvm/bin"


@pytest.mark.parametrize("source", ge.SOURCES)
def test_no_packed_float32_instructions(source, tmp_path):
    """Some of their forms have given wrong results on this part; the compiler makes them by itself unless told not to."""
    obj = os.path.join(ge.CSRC, source.replace(".hip", ".o"))
    if not os.path.exists(obj) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("no object file of this build, or no disassembler")
    bundle, code = str(tmp_path / "bundle"), str(tmp_path / "code.o")
    subprocess.run([os.path.join(LLVM, "llvm-objcopy"), "--dump-section=.hip_fatbin=" + bundle, obj, str(tmp_path / "copy.o")],
                   check=True)
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", "--unbundle", "--input=" + bundle,
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + code], check=True)
    text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", code], check=True, capture_output=True, text=True).stdout
    assert "s_endpgm" in text
    assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)


def test_build_compiles_whenever_it_is_called(monkeypatch):
    """Also where the libraries are newer than their sources: it is the check that the sources compile."""
    ran = []

    class Compiled:
        def wait(self):
            return 0

    monkeypatch.setattr(ge.subprocess, "Popen", lambda cmd, **k: ran.append(cmd[-1]) or Compiled())
    monkeypatch.setattr(ge.subprocess, "run", lambda cmd, **k: ran.append(cmd[-1]))
    ge.build()
    assert [os.path.basename(o) for o in ran[:len(ge.SOURCES)]] == [s.replace(".hip", ".o") for s in ge.SOURCES]
    assert len(ran) == len(ge.SOURCES) + 2                      # and the two links
