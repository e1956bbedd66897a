"""CPU tests: the batched operators of the beam search refuse missing pointers before they
touch a device."""
import ctypes

import pytest

import synapse_b200 as sb

L = sb.lib
ONE = ctypes.c_void_p(8)
F = ctypes.c_float(1e-6)


def test_null_pointers():
    p = ctypes.c_void_p()
    n = ctypes.c_size_t()
    assert L.syn_cuda_kvcache_pool(None, 0, ctypes.byref(p), ctypes.byref(p)) == 1
    assert L.syn_cuda_kvcache_page_table(None, ctypes.byref(p), ctypes.byref(n)) == 1
    assert L.syn_cuda_kvcache_fork(None, 0, 1, 4, None) == 1
    assert L.syn_cuda_kvcache_reorder(None, 2, ONE, ONE, 2, None) == 1
    assert L.syn_cuda_kvcache_reorder(ONE, 2, None, ONE, 2, None) == 1
    assert L.syn_cuda_kvcache_reorder(ONE, 2, ONE, None, 2, None) == 1
    assert L.syn_cuda_decode_plan_create(None, 4, ctypes.byref(p)) == 1
    assert L.syn_cuda_decode_plan_create(ONE, 4, None) == 1
    assert L.syn_cuda_decode_plan_destroy(None) == 1
    assert L.syn_cuda_decode_plan_set(None, 0, None, None, None) == 1
    assert L.syn_cuda_decode_plan_set(ONE, 1, None, ONE, None) == 1
    assert L.syn_cuda_decode_plan_prefix(None, 0, ctypes.byref(n)) == 1
    assert L.syn_cuda_generate_beam(None, 0, ONE, 1, 1, 1, -1, ONE, ONE) == 1
    assert L.syn_cuda_generate_beam(ONE, 0, None, 1, 1, 1, -1, ONE, ONE) == 1
    assert L.syn_cuda_generate_beam(ONE, 0, ONE, 1, 1, 1, -1, None, ONE) == 1


@pytest.mark.parametrize("missing", [0, 2, 3, 4, 9, 10, 12])
def test_attention_decode_shared_needs_its_arrays(missing):
    a = [ONE, 0, ONE, ONE, ONE, 64, None, None, F, ONE, ONE, 0, ONE, 64, None]
    a[missing] = None
    assert L.syn_cuda_attention_decode_shared(*a) == 1


@pytest.mark.parametrize("missing", [0, 3, 4, 5, 6, 7, 13, 14, 15])
def test_append_batch_needs_its_arrays(missing):
    a = [ONE, 0, 1, ONE, ONE, ONE, ONE, ONE, 64, 1, None, None, F, ONE, ONE, ONE, 64, None]
    a[missing] = None
    assert L.syn_cuda_qk_norm_rope_kv_append_batch(*a) == 1


def test_beam_select_checks_before_any_launch():
    def call(ctx=ONE, x=ONE, ld=10, groups=1, beams=2, vocab=10, s=ONE, fin=None, eos=-1, k=2, out=ONE):
        return L.syn_cuda_beam_select(ctx, x, ld, groups, beams, vocab, s, fin, eos, k, out, ONE, ONE,
                                      None, None)
    assert call(ctx=None) == call(x=None) == call(s=None) == call(out=None) == 1
    assert call(groups=0) == 0
    assert call(beams=0) == call(vocab=0) == call(k=0) == 7
    assert call(ld=9) == 4
    assert call(beams=65) == call(k=65, vocab=100, ld=100) == 12
    assert call(vocab=(1 << 25) + 1, ld=(1 << 25) + 1) == 12
    assert call(groups=40000) == 12  # 80000 rows
    assert call(beams=1, vocab=3, k=4) == 2
    assert call(fin=ONE, eos=-1) == call(fin=ONE, eos=10) == 2
