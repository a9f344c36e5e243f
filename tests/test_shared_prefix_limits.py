"""Shared prefixes: sizes past every limit at the C entries, which need no GPU."""

import subprocess
import sys
from pathlib import Path

import pytest

from aiproj_amd import _native

FP8, BF16, I32, I64 = _native.E4M3FN, _native.BF16, _native.I32, _native.I64
SOME = 4096          # an address that a refused call does not look at


@pytest.mark.parametrize("sizes", [(2 ** 62, 4, 4, 64, 1, 8, 16), (2 ** 61, 8, 8, 64, 1, 8, 16), (2 ** 60, 64, 80, 2, 2 ** 30, 2 ** 62, 2 ** 26),
                                   (2 ** 63 - 1, 2 ** 31 - 1, 1, 512, 0, 2 ** 63 - 1, 2 ** 31 - 1), (2 ** 40, 32, 8, 128, 1, 8, 16),
                                   (4, 8, 2, 64, 1, 2 ** 60, 16), (4, 8, 2, 64, 1, 2 ** 31, 1), (4, 8, 2, 513, 1, 8, 16)])
def test_workspace_of_sizes_past_the_limits(sizes):
    """Products of sizes that pass 64 bits end no process (asked for in one of its own), and what calls refuse needs nothing."""
    ask = "from aiproj_amd import _native; f = _native.lib().kvfp8_shared_prefix_workspace_bytes; " \
          f"print([f(*{sizes}, kv, prompt) for kv in range(4) for prompt in (0, 1)])"
    done = subprocess.run([sys.executable, "-c", ask], capture_output=True, text=True, cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0 and done.stdout.strip() == str([0] * 8)


@pytest.mark.parametrize("width,page,code", [(2 ** 60, 16, -6), (2 ** 59, 32, -6), (2 ** 62, 1, -6), (2 ** 27 - 512, 16, -6),
                                             (2 ** 27 - 513, 16, -5)])
def test_tables_whose_tokens_pass_64_bits_are_refused(width, page, code):
    lib = _native.lib()
    decode = lib.kvfp8_shared_prefix_decode(SOME, BF16, 256, 64, 1, 4, 2, 64, SOME, SOME, BF16, None, None, 8, page, SOME, 4, width,
                                            SOME, I64, SOME, I32, 0.1, SOME, None, 0, None, SOME, I64, SOME, I64, SOME, I64, 1)
    prefill = lib.kvfp8_shared_prefix_prefill(SOME, BF16, 2, 4, 2, 64, SOME, SOME, BF16, None, None, 8, page, SOME, 4, width, SOME,
                                              I64, SOME, I64, SOME, I64, 1, SOME, I32, 1, 2, 0.1, SOME, SOME, None, 0, None)
    assert decode == prefill == code


@pytest.mark.parametrize("rows,heads", [(2 ** 62, 4), (2 ** 32, 1), (2 ** 30, 4)])
def test_rows_past_32_bits_are_refused(rows, heads):
    prefill = _native.lib().kvfp8_shared_prefix_prefill(SOME, BF16, rows, heads, 1, 64, SOME, SOME, BF16, None, None, 8, 16, SOME, 4,
                                                        8, SOME, I64, SOME, I64, SOME, I64, 1, SOME, I32, 1, 2, 0.1, SOME, SOME, None,
                                                        0, None)
    assert prefill == -6
