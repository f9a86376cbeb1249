"""The paged write's second scale rule (amax times a reciprocal) under the quantizers'
three-operation quotient: the exhaustive host check of tests/pages_quotient_check.c."""
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.timeout(900)
def test_quotient_codes_equal_ieee_division_exhaustively(tmp_path):
    exe = tmp_path / "pages_quotient_check"
    subprocess.run(["gcc", "-O2", "-fopenmp", "-ffp-contract=off", "-fno-fast-math", "-o", str(exe),
                    str(ROOT / "tests" / "pages_quotient_check.c"), str(ROOT / "oracle" / "fp8_oracle.c"), "-lm"],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=880)
    print(out.stdout)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.count(" 0 code mismatches, 0 rows past") == 2
