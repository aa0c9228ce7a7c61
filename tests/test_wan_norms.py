"""Which norms the Wan hook's fused path takes (fused_norm_rope=True): RMS norms over all heads, each with its own epsilon, or none; anything else is
refused instead of being computed as something that it is not."""
import importlib.util
import os

import pytest
import torch

spec = importlib.util.spec_from_file_location("_hooks_cpu_for_norms", os.path.join(os.path.dirname(os.path.abspath(__file__)), "test_model_hooks_cpu.py"))
hooks_cpu = importlib.util.module_from_spec(spec)
spec.loader.exec_module(hooks_cpu)

HEADS, D, L, GRID = 2, 64, 30, (2, 3, 4)


class _Rms(torch.nn.Module):
    """An RMS norm of a model's own, its epsilon under one of the two usual names."""

    def __init__(self, dim, eps, name="eps"):
        super().__init__()
        self.weight = torch.nn.Parameter(1 + 0.2 * torch.randn(dim))
        if name:
            setattr(self, name, eps)


def block(norm_q, norm_k):
    from mpsa import model_hooks as H
    torch.manual_seed(0)
    model = hooks_cpu._Wan(dim=HEADS * D, heads=HEADS, n=1)
    att = model.blocks[0].self_attn
    att.norm_q, att.norm_k = norm_q, norm_k
    H.set_mpsa_attn_wan(model, fused_norm_rope=True)
    return model, att


def angles():
    ang = torch.arange(64, dtype=torch.float64)[:, None] * torch.cat([1e4 ** (-torch.arange(n, dtype=torch.float64) / n) for n in (12, 10, 10)])
    return torch.polar(torch.ones_like(ang), ang)


def call(att, device="cpu"):
    return att(torch.randn(1, L, HEADS * D, device=device), torch.tensor([L]), torch.tensor([GRID]), angles())


@pytest.fixture
def recorded(monkeypatch):
    """norm_rope is replaced by a recorder: what it is called with for queries (k None or not) and keys."""
    from mpsa import model_hooks as H, serving
    seen = []

    def norm_rope(q, k=None, **kw):
        seen.append((k is not None, kw["q_weight"], kw.get("k_weight"), kw["norm"], kw["across_heads"], kw["eps"]))
        return q if k is None else (q, k)

    monkeypatch.setattr(serving, "norm_rope", norm_rope)
    monkeypatch.setattr(H, "mxfp_kernel", lambda q, k, v, mask, **kw: v)
    return seen


W = HEADS * D


@pytest.mark.parametrize("norm_q,norm_k", [
    (torch.nn.LayerNorm(W), torch.nn.LayerNorm(W)), (_Rms(W, 1e-6), torch.nn.LayerNorm(W, bias=False)), (torch.nn.LayerNorm(W, elementwise_affine=False), torch.nn.Identity()),
    (torch.nn.RMSNorm(D), torch.nn.RMSNorm(D)), (torch.nn.RMSNorm(W, elementwise_affine=False), torch.nn.RMSNorm(W, elementwise_affine=False)),
    (_Rms(W, 0, name=None), _Rms(W, 0, name=None)), (torch.nn.GroupNorm(1, W), torch.nn.GroupNorm(1, W)), (torch.nn.Linear(W, W, bias=False), torch.nn.Identity()),
], ids=["layer norm", "layer norm without bias", "layer norm without weight", "each head", "no weight", "no epsilon", "group norm", "no norm"])
def test_other_norms_are_refused(recorded, norm_q, norm_k):
    _, att = block(norm_q, norm_k)
    with pytest.raises(ValueError):
        call(att)
    assert not recorded


def test_one_call_where_the_norms_are_alike(recorded):
    a, b = _Rms(W, 1e-5), _Rms(W, 1e-5, "variance_epsilon")
    call(block(a, b)[1])
    (both, wq, wk, norm, across, eps), = recorded
    assert both and wq is a.weight and wk is b.weight and norm and across and eps == 1e-5
    recorded.clear()
    call(block(torch.nn.Identity(), torch.nn.Identity())[1])
    (both, wq, wk, norm, across, eps), = recorded
    assert both and wq is None and wk is None and not norm


def test_each_norm_has_its_own_epsilon(recorded):
    a, b = _Rms(W, 1e-5), torch.nn.RMSNorm(W)                  # (none given: the type's)
    call(block(a, b)[1])
    assert [(x[0], x[1] is w, x[5]) for x, w in zip(recorded, (a.weight, b.weight))] == [(False, True, 1e-5), (False, True, torch.finfo(torch.float32).eps)]
    recorded.clear()
    call(block(a, torch.nn.Identity())[1])
    assert [(x[0], x[3]) for x in recorded] == [(False, True), (False, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [(1e-2, 1e-2), (1e-2, 1e-1), (None, None), (None, 0.5)])
def test_the_result_is_that_of_the_norms(eps):
    from test_gpu_serving import BF16, half_step
    torch.manual_seed(1)
    norms = [torch.nn.RMSNorm(W, eps=e) for e in eps]
    for n in norms:
        n.weight.data = 1 + 0.2 * torch.randn(W)
    model, att = block(*norms)
    model = model.cuda()
    seen = []

    class Recorder(torch.nn.Module):
        def forward(self, q, k, v, **kw):
            seen.append((q, k))
            return v

    att.inner_attention = Recorder()
    x = 0.3 * torch.randn(1, L, W, device="cuda")
    freqs = angles()
    att(x, torch.tensor([L]), torch.tensor([GRID]), freqs)
    f, h, w = GRID
    i = torch.arange(f * h * w)
    turn = torch.cat((freqs[i // (h * w), :12], freqs[i // w % h, 12:22], freqs[i % w, 22:]), 1)[None, :, None]
    for got, lin, norm, e in zip(seen[0], (att.q, att.k), (att.norm_q, att.norm_k), eps):
        y = lin(x).detach().double().cpu()
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + (torch.finfo(torch.float32).eps if e is None else e)) * norm.weight.detach().double().cpu()
        y = y.reshape(1, L, HEADS, D)
        z = torch.view_as_complex(y[:, :f * h * w].reshape(1, -1, HEADS, D // 2, 2).contiguous()) * turn
        y[:, :f * h * w] = torch.view_as_real(z).flatten(-2)
        # fp32 throughout (2^-24 of a few operations of elements of size 6 at most), then bf16
        assert bool(((got.double().cpu() - y).abs() <= half_step(BF16) * y.abs() * 1.01 + 2.0 ** -17).all())
