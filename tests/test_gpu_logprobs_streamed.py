"""token_logprobs where a row is read in several batches of elements, in every type.

A row (or slice) of more elements than a work-group holds at once, 8,192 in 16 bits and
4,096 in fp32, is streamed; rows enough to fill the chip are not cut into slices.  Here
600 rows of 20,000 or 9,000 logits, and 64 of 300,000, which are cut into slices that
are streamed.  Checks and tolerances are test_gpu_logprobs_magnitudes's.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from gpu_cases import DEV
from test_gpu_logprobs import logits_of
from test_gpu_logprobs_magnitudes import Rows, repeated

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIGNALLING = {torch.float32: 0x7F800001, torch.float16: 0x7C01, torch.bfloat16: 0x7F81}
QUIET = {torch.float32: 0x7FC00000, torch.float16: 0x7E00, torch.bfloat16: 0x7FC0}


def vocab_of(dtype):
    return 9000 if dtype == torch.float32 else 20000


def bits_of(x):
    return x.view(torch.int32 if x.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["signalling", "quiet"])
@pytest.mark.parametrize("late", [False, True])
def test_nan_beside_the_largest(gpu_ops, dtype, kind, late):
    """One NaN in each place of a 16-byte vector, the row's largest in each other place, in
    the first batch of elements and in a later one."""
    vocab, n = vocab_of(dtype), 16 // dtype.itemsize
    nan = (SIGNALLING if kind == "signalling" else QUIET)[dtype]
    at = vocab // n // 4 * 3 * n if late else 5 * n
    places = [(k, j) for k in range(n) for j in range(n) if k != j]
    x = logits_of(len(places), vocab, dtype, 8)
    for row, (k, j) in enumerate(places):
        bits_of(x)[row, at + k] = nan
        x[row, at + j] = 40.0
    repeated(gpu_ops, x, [at + j for _, j in places], 9, 600)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [0, 600])
def test_vectors_of_nan(gpu_ops, dtype, rows):
    """All of a vector but its largest NaN, whole vectors and chunks of them, alternating
    kinds, and NaN ahead of every chunk's largest; held in registers too (no ``rows``)."""
    vocab, n = vocab_of(dtype) if rows else 3000, 16 // dtype.itemsize
    x = logits_of(2 * n + 3, vocab, dtype, 9)
    bits, kinds = bits_of(x), (SIGNALLING[dtype], QUIET[dtype])
    top = vocab // 2 // n * n
    for j in range(n):
        for row, nan in ((j, kinds[0]), (n + j, kinds[1])):
            bits[row, top : top + n] = nan
            x[row, top + j] = 40.0
    bits[2 * n, : vocab // 2] = kinds[0]
    bits[2 * n + 1, 1::2] = kinds[0]
    bits[2 * n + 1, 3::4] = kinds[1]
    bits[2 * n + 2, 2::3] = kinds[0]
    tokens = [top + j % n for j in range(2 * n)] + [vocab - 1, 1, 0]
    if rows:
        repeated(gpu_ops, x, tokens, 64, rows)
    else:
        Rows(x, tokens, 64).run(gpu_ops).check()


def special_rows(vocab, dtype):
    info = torch.finfo(dtype)
    x = logits_of(16, vocab, dtype, 5)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, vocab - 1] = -3.0
    x[2, 5:] = -math.inf
    x[3] = info.min
    x[4] = info.min
    x[4, vocab // 2] = 1.0
    x[5, ::2] = math.nan
    x[6] = math.nan
    x[7, 3], x[7, vocab - 2] = math.inf, math.inf
    x[8] = 0.0
    x[8, ::3] = -0.0
    x[9] = info.max
    x[10] = -math.inf
    x[10, ::7] = 2.0
    x[11, 1:] = -30.0
    x[11, 0] = 30.0
    up = torch.arange(vocab, device=DEV) / vocab * 8
    x[12], x[13] = up, up.flip(0)
    x[14] = torch.arange(vocab, device=DEV) // 100 % 7 * 0.5
    x[15, : vocab * 4 // 5] = info.min
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_special_rows(gpu_ops, dtype, top):
    """No token, one, few, all equal, infinities, the type's lowest and largest values, zeros
    of both signs, ascending and descending rows."""
    vocab = vocab_of(dtype)
    rng = random.Random(top)
    tokens = [0, vocab - 1, 4, 1, vocab // 2, 1, 0, vocab - 2, 63, 9, 14, 0, vocab - 1, vocab // 3, 700, vocab - 1]
    repeated(gpu_ops, special_rows(vocab, dtype), tokens, top, 600)
    repeated(gpu_ops, special_rows(vocab, dtype), [rng.randrange(-1, vocab + 1) for _ in tokens], top, 600)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows_in_slices(gpu_ops, dtype):
    vocab = 300000
    tokens = [0, vocab - 1, 4, 1, vocab // 2, 1, 0, vocab - 2, 63, 9, 14, 0, vocab - 1, vocab // 3, 700, vocab - 1]
    repeated(gpu_ops, special_rows(vocab, dtype), tokens, 64, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [8193, 16384, 20003])
def test_odd_vocabularies(gpu_ops, dtype, vocab):
    """Rows that begin anywhere and end inside a vector, a chunk and a batch."""
    rng = random.Random(vocab)
    x = logits_of(21, vocab, dtype, vocab, pad=3)
    repeated(gpu_ops, x, [rng.randrange(-1, vocab + 1) for _ in range(21)], 20, 600)
