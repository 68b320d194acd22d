"""CPU checks of the packed-sequence operators: the kernels that the library holds, and calls that are decided on the host."""

import re

import pytest
import torch

from appcorr_amd import _lib
from appcorr_amd import kernels as K
from tests.test_packed_refusals import NULL, P16, norm_args, refused, rope_args


def test_every_attention_kernel_of_the_library_is_one_that_a_call_takes():
    """Rows kernels of 4 waves (128 rows), 8 only at Dh = 128; keys kernels of 4 waves, 8 only at Dh = 64; a merge for
    each height of a tile."""
    blob = _lib.LIB_PATH.read_bytes()

    def instances(kernel):
        found = re.findall(kernel.encode() + rb"INS_8Attn(Bf16|Fp16)E((?:Li\d+E)+)E", blob)
        return {(e.decode(), *map(int, re.findall(rb"\d+", n))) for e, n in found}

    def both(*shapes):
        return {(e, *s) for e in ("Bf16", "Fp16") for s in shapes}

    assert instances("packed_attn_rows_kernel") == both((64, 4), (128, 4), (128, 8))
    assert instances("packed_attn_keys_kernel") == both((64, 4), (64, 8), (128, 4))
    assert instances("packed_attn_merge_kernel") == both((64, 16), (64, 128), (128, 16), (128, 128), (128, 256))


@pytest.mark.parametrize("kw", [dict(B=0), dict(N=0), dict(B=0, N=0, kv_bs=0)])
def test_a_cache_without_slots_skips_every_row(kw):
    """Nothing is launched, and torch gives an empty cache no address; other arguments are checked all the same."""
    host, args = norm_args(kv=NULL, **kw)
    _lib.call("oudjat_qk_norm_rope_kv", *args)
    host, args = norm_args(kv=NULL, qo_rs=0, **kw)
    refused("OUDJAT_ERR_UNSUPPORTED_LAYOUT", "oudjat_qk_norm_rope_kv", *args)
    host, args = norm_args(kv=NULL)
    refused("OUDJAT_ERR_INVALID_ARGUMENT", "oudjat_qk_norm_rope_kv", *args)


def test_sections_are_whole_numbers():
    """Fractions were cut one by one, and inv_freq checked against their sum: (4.5, 4.5) took 9 frequencies and read 8."""
    pos = torch.zeros(3, 2)
    for sections, count in (((4.5, 4.5), 9), ((7.5, 8.5), 16)):
        with pytest.raises(ValueError, match="whole numbers"):
            K._axis_rope(pos, torch.zeros(count), sections, 3, "rope")
    for sections in ((16, 16), [16, 16], (16.0, 16.0), torch.tensor([16, 16])):
        assert K._axis_rope(pos, torch.zeros(32), sections, 3, "rope")[4] == 2


def test_rope_refuses_one_output_for_q_and_k():
    """In place with q for both, say: each head would be turned by two threads, once or twice."""
    host, args = rope_args(qo=P16, ko=P16)
    refused("OUDJAT_ERR_INVALID_ARGUMENT", "oudjat_rope_axes", *args)
    host, args = rope_args(rows=0, qo=P16, ko=P16)
    _lib.call("oudjat_rope_axes", *args)


def test_a_cpu_tensor_has_no_stream():
    """Its device index, -1, is the current device to torch: a launch with the tensor's address would follow."""
    with pytest.raises(ValueError, match="GPU tensor"):
        _lib.stream_of(torch.zeros(1))
