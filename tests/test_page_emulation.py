"""The page-cache and rotary kernels on the CPU: their own per-workgroup code, with host threads as lanes, on buffers of
exactly the size they may touch, under the sanitizers (tests/cpp/page_sweep.cc); and what the entry points refuse before
they need a GPU."""
import ctypes as C
import os
import subprocess

import pytest

import multimesh_jax_amd as mm
from multimesh_jax_amd import _binding as B

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("program,rounds", [("page_sweep", 60), ("page_sweep_threads", 20)])
def test_kernels_under_the_sanitizers(program, rounds):
    p = subprocess.run([os.path.join(HERE, "cpp", program), str(rounds)], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0 and p.stdout.strip().endswith("OK"), p.stdout + p.stderr


def test_null_arguments():
    lib = mm.load()
    out = C.c_void_p()
    options = B.RotaryOptions(rotary_dim=8, base=10000.0, magnitude=1.0)
    calls = [
        lambda: lib.mmr_pages_create(None, None, 0, None, None, None, 1, C.byref(out)),
        lambda: lib.mmr_pages_destroy(None), lambda: lib.mmr_pages_extend(None, None, None, 0),
        lambda: lib.mmr_pages_fork(None, None, None, 0), lambda: lib.mmr_pages_free(None, None, 0),
        lambda: lib.mmr_pages_copy(None, None, None, 0), lambda: lib.mmr_pages_compact(None),
        lambda: lib.mmr_pages_status(None, None, None),
        lambda: lib.mmr_pages_write(None, None, None, 0, 0, None, -1, None, None, None, None),
        lambda: lib.mmr_rotary_create(None, C.byref(options), C.byref(out)), lambda: lib.mmr_rotary_destroy(None),
        lambda: lib.mmr_rotary_apply(None, None, None, 0, None, 0, 0),
    ]
    for call in calls:
        assert call() == 1  # MMR_INVALID_ARGUMENT
        assert b"null" in lib.mmr_last_error()


def test_options_layout_matches_the_header():
    import tempfile
    src = '#include <stdio.h>\n#include "mmreshard.h"\nint main(void) { printf("%zu\\n", sizeof(mmr_rotary_options)); return 0; }'
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-std=c11", "-I", os.path.join(os.path.dirname(HERE), "include"), c, "-o", exe])
        assert int(subprocess.check_output([exe])) == C.sizeof(B.RotaryOptions)
