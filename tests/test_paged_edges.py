"""The paged operators and rotary_qk at their edges, without a GPU: what the C entry points
refuse, and what the operators' own Python code does around a kernel (a stand-in here)."""

import pytest
import torch

import mrsa
from mrsa import _lib, paged_cache, rotary


def test_c_append_without_kv_heads_still_needs_its_table():
    s = (512, 512, 128)
    status = _lib.call("mrsa_paged_append_fwd", 4096, *s, None, 0, 0, 0, None, 0, 0, 0, None, None, 0,
                       None, 0, 0, 4096, 1, 1, None, 4, 4, 7, 16, None, *s, None, *s, 1, 1, 4, 0,
                       128, 0, 0, 0, 4096, None)
    assert status == _lib.MRSA_ERR_INVALID_ARGUMENT


@pytest.fixture
def cpu_ops(monkeypatch):
    """The operators' own code on CPU tensors, with a stand-in for the library: what it was
    called with is kept, nothing is computed."""

    calls = []

    def call_on(device, name, *args):
        calls.append(name)
        return _lib.MRSA_OK

    monkeypatch.setattr(_lib, "call_on", call_on)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(paged_cache, "check_heads", lambda t, name: None)
    monkeypatch.setattr(rotary, "check_heads", lambda t, name: None)
    lib = torch.library.Library("mrsa", "IMPL")
    lib.impl("paged_append_", paged_cache._paged_append_impl, "CPU")
    lib.impl("paged_attention", paged_cache._paged_attention_impl, "CPU")
    lib.impl("copy_pages_", paged_cache._copy_pages_impl, "CPU")
    yield calls
    lib._destroy()


def _pools(**kw):
    return torch.zeros(2, 5, 16, 2, 64, **kw), torch.zeros(2, 5, 16, 2, 64, **kw)


def _append(kp, vp, **kw):
    k = torch.zeros(1, 3, 2, 64)
    mrsa.paged_cache_append(k, k, kp, vp, torch.zeros(1, 5, dtype=torch.int32),
                            torch.arange(3)[None], **kw)


def test_in_place_operators_raise_the_pools_version_counters(cpu_ops):
    # (what torch itself goes by to refuse a stale backward pass, and kv_fragments_cached to lay
    # a changed K / V out again)
    kp, vp = _pools()
    view = kp[0].view(1, 80, 2, 64)
    before = kp._version, vp._version, view._version
    _append(kp[0], vp[0])
    after = kp._version, vp._version, view._version
    assert all(b > a for a, b in zip(before, after))
    torch.ops.mrsa.copy_pages_(kp, vp, [0], [1])
    assert kp._version > after[0] and vp._version > after[1] and view._version > after[2]
    w = torch.ones(2, 5, 16, 2, 64, requires_grad=True)
    loss = (w * kp).sum()
    _append(kp[1], vp[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():       # those tensors have no counter
        kp, vp = _pools()
    _append(kp[0], vp[0])
    torch.ops.mrsa.copy_pages_(kp, vp, [0], [1])
    assert cpu_ops == ["mrsa_paged_append_fwd", "mrsa_copy_pages",
                       "mrsa_paged_append_fwd", "mrsa_paged_append_fwd", "mrsa_copy_pages"]
