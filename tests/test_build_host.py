"""The build scripts: no HIP source is compiled without the flag against two-wide float32 instructions, and what the shipped
library is made of is checked for them."""
import glob
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero_gomoku_amd", "csrc")
KERNEL = "%s:\n\tv_add_f32 v0, v1, v2\n%s\ts_endpgm\n\t.amdhsa_kernel %s\n"


def commands(path):
    text = open(path).read().replace("\\\n", " ")
    return [l for l in text.splitlines() if not l.lstrip().startswith("#") and "hipcc" in l and ".hip\"" in l]


@pytest.mark.parametrize("script", sorted(glob.glob(os.path.join(CSRC, "*.sh"))))
def test_every_compilation_has_the_flag(script):
    text = open(script).read()
    for line in commands(script):
        assert "$nopk" in line, line
        assert 'nopk="-Xclang -target-feature -Xclang -packed-fp32-ops"' in text


def test_the_build_checks_every_source_it_compiles():
    build = os.path.join(CSRC, "build.sh")
    sources = {os.path.basename(p)[:-4] for p in glob.glob(os.path.join(CSRC, "*.hip"))}
    check = [l for l in open(build).read().splitlines() if "check_asm.sh\"" in l]
    assert len(check) == 1
    for name in sources:
        assert any("/%s.hip\"" % name in l for l in commands(build)) and "/%s*gfx950.s" % name in check[0], name


@pytest.mark.parametrize("name", ["_ZN3azg13search_kernelEv", "_ZN6azgops11fix_kernelEv"])
def test_check_asm(tmp_path, name):
    def run(*texts):
        files = []
        for i, t in enumerate(texts):
            files.append(str(tmp_path / ("%d.s" % i)))
            open(files[-1], "w").write(t)
        r = subprocess.run(["sh", os.path.join(CSRC, "check_asm.sh")] + files, capture_output=True, text=True)
        return r.returncode, r.stderr
    clean = KERNEL % (name, "", name)
    assert run(clean, clean) == (0, "")
    for op in ("v_pk_fma_f32 v[0:1], v[2:3], v[4:5], v[6:7]", "v_pk_mul_f32 v[0:1], v[2:3], v[4:5]", "v_pk_add_f32 v[0:1], v[2:3], v[4:5]"):
        rc, text = run(clean, KERNEL % (name, "\t" + op + "\n", name))
        assert rc == 1 and name in text and op.split()[0] in text
    assert run()[0] == 1 and run("")[0] == 1
    assert subprocess.run(["sh", os.path.join(CSRC, "check_asm.sh"), str(tmp_path / "none.s")], capture_output=True).returncode == 1
