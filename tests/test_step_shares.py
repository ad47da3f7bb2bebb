"""The arithmetic of tokens' shares (csrc/gv_shares.h) on the host, against long double."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_shares(tmp_path):
    probe = tmp_path / "probe"
    subprocess.run(["g++", "-O2", "-std=c++17", "-mfma", "-o", str(probe), os.path.join(ROOT, "tests", "shares_probe.cpp")], check=True)
    table, rest, finely, with_whole, whole, ends, wide, order = subprocess.run([str(probe)], check=True, capture_output=True, text=True).stdout.split()
    assert float(table) <= -53  # half a step
    # a^5 / 1920 = 2^-43.5 at a = ln 2 / 64; a little beyond it (a whole part from 32 bits is off by 2^-8 at most: 0.505 for 0.5) 1 % more in a is
    # 5 % more in a^5, and the sixth term of the series a^6 / 720 = 2^-48.6: 2^-43.1
    assert float(rest) <= -43.1
    # 1.4e-16 (2^-52.7) and two roundings of 1.1e-16 (2^-53) of numbers near one are 3.6e-16
    assert float(finely) <= -51.3
    # with the table's 2^-53, the exponent's rounding (2^-53 of at most 2^8 octaves * ln 2: 2^-45.5) and three roundings: 2^-42.8
    assert float(with_whole) <= -42.8 and float(whole) <= -42.8
    assert ends == wide == order == "1"
