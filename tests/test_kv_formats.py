"""What the header says of the 4-bit format of a K/V cache: how far an element may be off,
where that ends, and how many bytes a row takes. On the CPU."""
import os
import subprocess

import numpy as np
import pytest

import pages_ref as pref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mormot2-qwen-tts_amd")


def rows_of(rng, most, n, hd):
    """Rows whose largest is `most`, some groups of them far smaller or zero."""
    x = rng.standard_normal((n, hd // 32, 32)) * np.exp(2 * rng.standard_normal((n, hd // 32, 1)))
    x[::5, 0] = 0
    x = x.reshape(n, hd)
    x *= most / np.abs(x).max(-1, keepdims=True)
    return x.astype(np.float32)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("most", [1e-44, 1.2e-42, 1.4e-42, 1e-41, 1e-38, 2.2e-35, 1e-30, 1e-3, 1.0,
                                  7.0, 1785.0, 3.3e38])
def test_elements_of_four_bits_are_as_near_as_said(most, hd):
    """Half a step, step * scale / 2 <= max of the 32 / 14 + scale / 2, and scale is the
    row's largest / 1785. Beside it the scale rounded to f32, by 2^-24 of it, or 2^-150 of
    a subnormal one, which leaves the row's largest as much of itself, or 1785 * 2^-150 <
    1.26e-42, above 7 * 255 scales; and the product rounded to f32, by 2^-24 of the element:
    together 2^-23 of the row's largest, where it is below 2.2e-35 (a subnormal scale)
    1.26e-42 + 2^-24 * 2.2e-35 < 2.6e-42."""
    x = rows_of(np.random.default_rng(hd), most, 2000, hd)
    off = np.abs(pref.stored(x, pref.Q4).astype(np.float64) - x.astype(np.float64))
    wide = np.abs(x.astype(np.float64))
    group = np.repeat(wide.reshape(len(x), -1, 32).max(-1), 32, -1)
    row = wide.max(-1, keepdims=True)
    assert (off <= group / 14 + row / 3570 + np.maximum(2.0 ** -23 * row, 2.6e-42)).all()
    # (and not far less: the bound is one that rows come to)
    if most > 1e-40:
        assert (off / (group / 14 + row / 3570)).max() > 0.9


def test_rows_below_a_normal_scale():
    """A scale of up to 2^-150 rounds to zero, and with it the row."""
    x = rows_of(np.random.default_rng(1), 1.2e-42, 100, 64)
    assert not pref.stored(x, pref.Q4).any() and x.any()
    x = rows_of(np.random.default_rng(2), 1.4e-42, 100, 64)
    assert pref.stored(x, pref.Q4).any()
    # 2.2e-35 / 1785 is a normal number, 2.0e-35 / 1785 is not
    tiny = np.finfo(np.float32).tiny
    assert np.float32(2.2e-35 / 1785) >= tiny > np.float32(2.0e-35 / 1785)


def test_bytes_of_a_row(tmp_path):
    source = r"""
#include <cstdio>
#include "q3h_draft.h"
int main() {
  for (int hd : {64, 128})
    std::printf("%zu %zu\n", q3h::kv_bytes(Q3H_KV_Q4, 1, 1, 1, hd),
                q3h::kv_bytes(Q3H_KV_Q4, 3, 5, 7, hd));
}
"""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = str(tmp_path / "bytes.hip"), str(tmp_path / "bytes")
    with open(src, "w") as f:
        f.write(source)
    subprocess.run([hipcc, "-O1", "-std=c++17", "--offload-host-only", "-I",
                    os.path.join(ROOT, "include"), "-I", os.path.join(PKG, "csrc"), src, "-o", exe],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60, check=True).stdout
    got = [int(x) for x in out.split()]
    # a position of a kv head: a key and a value
    assert got == [n for hd in (64, 128) for n in (2 * (hd // 2 + 8), 2 * 3 * 5 * 7 * (hd // 2 + 8))]
