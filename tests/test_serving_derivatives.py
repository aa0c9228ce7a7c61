"""Operands that ask for a derivative are refused by the serving calls, tangents of forward mode and rotary tables among them."""
import os
import sys

import pytest
import torch
import torch.autograd.forward_ad as fwAD

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def test_what_asks_for_a_derivative():
    from mpsa.serving import _no_gradient
    x, w = torch.randn(3), torch.randn(3, requires_grad=True)
    _no_gradient(x, None)
    for no_grad in (False, True):
        with torch.set_grad_enabled(not no_grad):
            if no_grad:
                _no_gradient(x, w)
            else:
                with pytest.raises(ValueError):
                    _no_gradient(x, w)
            with fwAD.dual_level():
                _no_gradient(x)
                with pytest.raises(ValueError):                # (torch.no_grad() leaves forward mode on)
                    _no_gradient(x, None, fwAD.make_dual(x, x))


@pytest.mark.gpu
@pytest.mark.parametrize("long_way", [False, True])
def test_tangents_and_tables_are_refused(long_way, monkeypatch):
    import mpsa
    from mpsa import _lib
    if long_way:
        monkeypatch.setattr(_lib, "_native", _lib._LongWay)
    x = torch.ones(1, 2, 3, 64, dtype=torch.bfloat16, device="cuda")
    cos, sin, w = (torch.ones(8, 32, device="cuda"), torch.ones(8, 32, device="cuda"), torch.ones(64, device="cuda"))
    c = mpsa.kv_cache(2, 2, 64)
    table, i = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    with fwAD.dual_level():
        d, e, f = (fwAD.make_dual(t, torch.ones_like(t)) for t in (x, w, cos))
        for call in (lambda: mpsa.norm_rope(d), lambda: mpsa.norm_rope(x, d), lambda: mpsa.norm_rope(x, q_weight=e), lambda: mpsa.norm_rope(x, x, k_weight=e),
                     lambda: mpsa.norm_rope(x, rope=(f, sin)), lambda: mpsa.norm_rope(x, rope=(cos, f)), lambda: mpsa.kv_cache_append(c, d, x, table, i),
                     lambda: mpsa.kv_cache_append(c, x, d, table, i), lambda: mpsa.kv_cache_attention(d, c, table, i + 3)):
            with pytest.raises(ValueError):
                call()
        mpsa.norm_rope(x, x, q_weight=w, rope=(cos, sin))
    assert not c.k.any()
    f = cos.clone().requires_grad_()
    for rope in ((f, sin), (cos, f)):
        with pytest.raises(ValueError):
            mpsa.norm_rope(x, rope=rope)
        with torch.no_grad():
            assert torch.equal(mpsa.norm_rope(x, rope=rope), mpsa.norm_rope(x, rope=(cos, sin)))
