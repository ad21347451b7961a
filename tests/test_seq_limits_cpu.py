"""Limits of the operators over sequences that are seen without a GPU: shapes whose indices would not fit, and workspace sizes."""
import ctypes

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
