"""Random calls over the whole range of the 8-bit and the bounded KV cache's operators, against the fp64 oracle, with the
checks and the derived bounds of test_gpu_fp8_cache.py and test_gpu_kv_evict.py."""
import numpy as np
import pytest
import torch

from tests import test_gpu_fp8_cache as fp8
from tests import test_gpu_kv_evict as bounded

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _size(rng, lo, hi):
    return int(round(float(np.exp(rng.uniform(np.log(lo), np.log(hi))))))


def _heads(rng, most):
    hkv = _size(rng, 1, most)
    return hkv * _size(rng, 1, max(2, 70 // hkv)), hkv


def _lengths(rng, B, cap):
    return [int(rng.choice([0, 1, cap, cap + 7, int(rng.integers(0, cap + 1)), int(rng.integers(0, cap + 1))])) for _ in range(B)]


def _cache(rng):
    """block, page (0: padded), capacity"""
    block = 1 << int(rng.integers(4, 9))
    page = 0 if rng.random() < 0.5 else max(block, 1 << int(rng.integers(4, 9)))
    unit = page or block
    return block, page, unit * _size(rng, 1, max(1, 1500 // unit))


@pytest.mark.parametrize("seed", range(30))
def test_append(seed):
    rng = np.random.default_rng(1000 + seed)
    block, page, cap = _cache(rng)
    B, H, D, n = _size(rng, 1, 9), _size(rng, 1, 12), 16 * int(rng.integers(1, 9)), _size(rng, 1, 400)
    fp8._append(rng, _lengths(rng, B, cap), H, D, cap, block, page, n, TYPES[seed % 3])


@pytest.mark.parametrize("seed", range(30))
def test_decode(seed):
    rng = np.random.default_rng(2000 + seed)
    block, page, cap = _cache(rng)
    B, (Hq, Hkv), D = _size(rng, 1, 80), _heads(rng, 8), 16 * int(rng.integers(1, 9))
    c = fp8._decode_case(rng, _lengths(rng, B, cap), Hq, Hkv, D, block, page, TYPES[seed % 3], cap)
    fp8._check(c, *fp8._run_decode(c))


@pytest.mark.parametrize("seed", range(45))
def test_weights(seed):
    rng = np.random.default_rng(3000 + seed)
    dtype = TYPES[seed % 3]
    codes = [0, 0, 16, 32, 64][int(rng.integers(0, 5))]
    B, (Hq, Hkv) = _size(rng, 1, 4), _heads(rng, 6)
    D = 16 * int(rng.integers(1, 9)) if codes else int(rng.integers(1, 17)) * 8 if dtype != torch.float32 else int(rng.integers(1, 33)) * 4
    S = _size(rng, 1, 1200)
    S = -(-S // codes) * codes if codes else S
    L = 1 if seed % 4 == 0 else _size(rng, 1, 90)
    causal = bool(rng.random() < 0.6)
    q_offset = int(rng.integers(-L, S + 1)) if causal else 0
    lengths = None if rng.random() < 0.4 else _lengths(rng, B, S)
    bounded._check_weights(rng, B, Hq, Hkv, L, S, D, dtype, codes, lengths=lengths, causal=causal, q_offset=q_offset,
                           scale=None if rng.random() < 0.7 else float(rng.normal() * 0.2))


@pytest.mark.parametrize("seed", range(30))
def test_evict(seed):
    rng = np.random.default_rng(4000 + seed)
    scale_block = 0 if seed % 3 else 1 << int(rng.integers(4, 7))
    block = scale_block << int(rng.integers(0, 3)) if scale_block else 1 << int(rng.integers(0, 6)) if rng.random() < 0.5 else 1
    S = _size(rng, 1, 5000)
    S = -(-S // block) * block if scale_block else S
    recent = block * _size(rng, 1, max(1, S // block))
    keep = recent + block * int(rng.integers(0, max(1, S // block)))
    dtype = torch.float8_e4m3fn if scale_block else TYPES[int(rng.integers(0, 3))]
    B, H, D = _size(rng, 1, 5), _size(rng, 1, 9), 16 * int(rng.integers(1, 9))
    w = np.exp(rng.standard_normal((B, H, S))).astype(np.float32)
    if seed % 5 == 0:
        w = np.round(w)  # many ties
    bounded._evict(rng, B, H, S, D, _lengths(rng, B, S), keep, recent, block, dtype, scale_block, w)
