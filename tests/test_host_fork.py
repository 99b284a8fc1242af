"""lmc_model_fork_seq's page accounting on the CPU (tests/host_fork.c), under
AddressSanitizer and UndefinedBehaviorSanitizer: shared pages are taken once,
a writer of a shared page takes a copy, pages return to the pool with their
last holder, a pool that is short refuses the whole call."""
import os
import subprocess

import pytest

from lmc_b200 import synth

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SAN = ["-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-g", "-O1"]


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("fork"))
    lay = os.path.join(d, "layout.c")
    with open(lay, "w") as f:  # the struct's layout as the internal header has it
        f.write('#include <stddef.h>\n#include "%s"\n' % os.path.join(ROOT, "lmc_b200", "csrc", "lmc_internal.h"))
        f.write("const size_t qt_layout[5] = {offsetof(struct lmc_qtensor, rows), offsetof(struct lmc_qtensor, bytes), "
                "offsetof(struct lmc_qtensor, tiled), offsetof(struct lmc_qtensor, gemm_wscale), sizeof(struct lmc_qtensor)};\n")
    inc = ["-I/usr/local/cuda/include"]
    objs = []
    for src, flags in ((os.path.join(ROOT, "lmc_b200", "host", "lmc_model.c"), ["-std=c99"] + inc), (lay, inc),
                       (os.path.join(HERE, "host_fork.c"), [])):
        o = os.path.join(d, os.path.basename(src) + ".o")
        subprocess.check_call(["gcc"] + flags + SAN + ["-c", src, "-o", o])
        objs.append(o)
    exe = os.path.join(d, "fork")
    subprocess.check_call(["gcc"] + SAN + ["-o", exe] + objs + ["-lm", "-lpthread"])
    return exe


def test_fork_page_accounting(driver, tmp_path):
    path = synth.make_llama(str(tmp_path / "p.gguf"), L=2, D=64, H=4, Hkv=2, F=128, S=64, V=64, seed=1)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1")
    r = subprocess.run([driver, path], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    steps = [tuple(int(v) for v in ln.split()[1:]) for ln in r.stdout.splitlines() if ln.startswith("F ")]
    launch, ok, oom, invalid = -2, 0, -4, -1
    assert steps == [(launch, 5), (ok, 5), (ok, 5), (ok, 5), (launch, 3), (launch, 3), (launch, 1), (ok, 2), (launch, 2),
                     (ok, 2), (oom, 2), (ok, 2), (ok, 5), (ok, 5), (ok, 8), (ok, 8), (invalid, 8), (invalid, 8), (invalid, 8)]
    assert "C -2 model_fork_seq: the model's KV cache is not paged" in r.stdout
