"""The paged operators and rotary_qk at their edges, without a GPU: what the C entry points
refuse, and what the operators' own Python code does around a kernel (a stand-in here)."""

from mrsa import _lib


def test_c_append_without_kv_heads_still_needs_its_table():
    s = (512, 512, 128)
    status = _lib.call("mrsa_paged_append_fwd", 4096, *s, None, 0, 0, 0, None, 0, 0, 0, None, None, 0,
                       None, 0, 0, 4096, 1, 1, None, 4, 4, 7, 16, None, *s, None, *s, 1, 1, 4, 0,
                       128, 0, 0, 0, 4096, None)
    assert status == _lib.MRSA_ERR_INVALID_ARGUMENT
