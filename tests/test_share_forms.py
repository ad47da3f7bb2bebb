"""Which form tokens' shares are worked out in (csrc/gv_shares.h), on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_plain_form_at_every_temperature(tmp_path):
    """Where it is taken its shares are shares: right to 2^-42.8 (tests/test_step_shares.py) down to 2^-200 of the largest, and next to nothing below."""
    probe = tmp_path / "probe"
    subprocess.run(["g++", "-O2", "-std=c++17", "-mfma", "-o", str(probe), os.path.join(ROOT, "tests", "share_forms_probe.cpp")], check=True)
    worst, below, ordinary, in_range, fitting = subprocess.run([str(probe)], check=True, capture_output=True, text=True).stdout.split()
    assert float(worst) <= -42.8 and float(below) <= -199 and ordinary == in_range == "1" and int(fitting) > 5000


def test_bins_of_ranges_of_any_extent(tmp_path):
    """Later bins for smaller values, the first for the largest, all bins in use where the range has an ordinary extent."""
    probe = tmp_path / "probe"
    subprocess.run(["g++", "-O2", "-std=c++17", "-mfma", "-o", str(probe), os.path.join(ROOT, "tests", "bins_probe.cpp")], check=True)
    assert subprocess.run([str(probe)], check=True, capture_output=True, text=True).stdout.split() == ["1"] * 4
