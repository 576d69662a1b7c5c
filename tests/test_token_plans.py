"""The token losses' plans, on the CPU: tests/plan_check/token_check builds the library's own host code and looks at what each
call of random shapes and limits of kept logits would run."""
import os
import subprocess

import pytest

from predicitivecoding_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def token_check(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("token_check") / "token_check")
    # the products' launchers are never called here, so their units are not built
    res = subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *build.HIPCC_FLAGS, "-O1", "-x", "hip",
                          os.path.join(HERE, "plan_check", "token_check.hip"), "-o", out,
                          "-Wl,--unresolved-symbols=ignore-all"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    return out


def run(exe, *args):
    res = subprocess.run([exe, *map(str, args)], capture_output=True, text=True, timeout=120)
    return res.returncode, res.stdout


@pytest.mark.parametrize("dtype,rows,dim,vocab,keep", [
    (2, 64, 784, 10000, 64 * 8 * 10048), (2, 64, 784, 10000, 5200000), (2, 64, 784, 10000, 64 * 8 * 10240 - 1),
    (1, 40, 64, 300, 200000), (1, 33, 520, 1315, 64 * 8 * 1344), (1, 64, 64, (1 << 20) + 70, 64 * 8 * ((1 << 20) + 128))])
def test_gradients_in_two_parts_keep_every_logit(token_check, dtype, rows, dim, vocab, keep):
    """A limit that the logits of whole 64s fit, and those of whole pieces do not."""
    rc, out = run(token_check, dtype, rows, dim, vocab, keep)
    assert rc == 0 and "stack 64" in out, out


@pytest.mark.parametrize("seed", [1, 2])
def test_random_losses_write_all_rows_of_their_gradients(token_check, seed):
    rc, out = run(token_check, seed, 30000)
    assert rc == 0, out[-2000:]
    assert int(out.split("plans, ")[1].split()[0]) > 5000, out
