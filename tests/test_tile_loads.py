"""CPU: the prompt and tree kernels' loads leave nothing to the scalar offset, from the code
the compiler wrote (voltattn_amd/libvoltattn_hip.so). A tile's rows past a prompt's or a
context's end read as zeros because the buffer descriptor ends there. Its range check is
documented for the vector and the immediate offset: a scalar one, above a short tile's size,
would leave the zeros to what the hardware does beyond that."""
import re
import subprocess

from tests.test_kernel_resources import LLVM, _code_objects


def test_loads_have_no_scalar_offset(tmp_path):
    seen, to_lds, bad = set(), 0, set()
    for i, obj in enumerate(_code_objects()):
        f = tmp_path / f"{i}.co"
        f.write_bytes(obj)
        with subprocess.Popen([LLVM + "objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", str(f)],
                              stdout=subprocess.PIPE, text=True) as p:
            name = ""
            for line in p.stdout:
                if line.endswith(">:\n"):
                    name = line.strip("<>:\n")
                elif ("prefill_causal" in name or "tree_attend" in name) and "buffer_load" in line:
                    soffset = re.search(r"s\[\d+:\d+\], (\S+)", line).group(1).rstrip(",")
                    seen.add(name)
                    to_lds += " lds" in line
                    if soffset != "0":
                        bad.add((name, line.strip()))
    assert len(seen) > 40 and to_lds > 0, (len(seen), to_lds)
    assert not bad, sorted(bad)[:4]
