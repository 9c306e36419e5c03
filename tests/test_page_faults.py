"""The page operators on the CPU, with host threads as lanes and under the sanitizers, on tables that are out of step with
themselves: one fault a case, the exact status and what is left (tests/cpp/page_faults.cc)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("program", ["page_faults", "page_faults_threads"])
def test_tables_out_of_step(program):
    p = subprocess.run([os.path.join(HERE, "cpp", program)], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0 and p.stdout.strip().endswith("OK"), p.stdout + p.stderr
