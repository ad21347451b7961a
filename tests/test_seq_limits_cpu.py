"""Limits of the operators over sequences that are seen without a GPU: shapes whose indices would not fit, and workspace sizes."""
import ctypes
import random

import pytest

from unet_amd import capi

QUERIES = [capi.unet_dot_attention_workspace_bytes, capi.unet_dot_attention_backward_workspace_bytes]


def need(f, num_seqs, total_q, total_k, heads_q, heads_kv, dim):
    n = ctypes.c_size_t(1 << 60)
    f(num_seqs, total_q, total_k, heads_q, heads_kv, dim, ctypes.byref(n))
    return n.value


@pytest.mark.parametrize("f", QUERIES)
@pytest.mark.parametrize("heads_q,heads_kv,dim", [(1 << 24, 1, 128), (1 << 25, 1, 64), (1 << 27, 1 << 10, 16), (3 << 23, 1 << 23, 100)])
def test_a_token_of_2_31_elements_is_refused(f, heads_q, heads_kv, dim):
    """The kernels count a token's elements in 32 bits: head h begins at element h * head_dim."""
    for total_q in (0, 1):
        with pytest.raises(RuntimeError, match="heads of"):
            need(f, 1, total_q, 1, heads_q, heads_kv, dim)
    need(f, 1, 1, 1, ((1 << 31) - 1) // dim, 1, dim)  # the most that fit


@pytest.mark.parametrize("f", QUERIES)
def test_token_counts_near_64_bits_are_refused(f):
    for total_q, total_k in ((2 ** 63 - 1, 1), (1, 2 ** 63 - 1), (2 ** 62, 2 ** 62)):
        with pytest.raises(RuntimeError, match="too many"):
            need(f, 1, total_q, total_k, 8, 2, 64)


@pytest.mark.parametrize("f", QUERIES)
def test_a_workspace_does_for_every_smaller_call(f):
    """Fewer tokens are cut into more shares, but a program that asks once, for its largest batch, has enough for all."""
    assert need(f, 1, 8192, 8192, 8, 8, 64) <= need(f, 1, 65536, 65536, 8, 8, 64)
    assert need(f, 4, 4, 65536, 32, 4, 128) <= need(f, 64, 64, 640000, 32, 4, 128)
    rng = random.Random(5)
    for _ in range(3000):
        heads_kv = rng.choice([1, 2, 3, 4, 8, 16])
        heads_q, dim = heads_kv * rng.choice([1, 2, 5, 8]), rng.choice([1, 16, 33, 64, 80, 100, 128])
        large = [rng.choice([1, 2, 7, 64, 300]), int(2 ** rng.uniform(0, 18)), int(2 ** rng.uniform(0, 18))]
        small = [rng.choice([1, 2, 7, 64, 300]), int(large[1] * rng.random()), int(large[2] * rng.random())]
        assert need(f, *small, heads_q, heads_kv, dim) <= need(f, *large, heads_q, heads_kv, dim), (large, small, heads_q, heads_kv, dim)


def test_workspaces_do_not_grow_without_end():
    # 2^15 rows of dim + 2 numbers; and two numbers a row and 3 * 2^16 rows of dK and dV
    assert need(QUERIES[0], 1, 10 ** 6, 10 ** 6, 8, 8, 128) <= 2 ** 15 * 130 * 4
    assert need(QUERIES[1], 1, 10 ** 6, 10 ** 6, 8, 8, 128) <= 8 * 8 * 10 ** 6 + 3 * 2 ** 16 * 2 * 128 * 4
