"""What the entries that serve a model token by token refuse before any GPU is touched, and the layout of their argument blocks."""
import ctypes

import pytest
import torch


def _call(name, args):
    from mpsa import _lib
    rc = getattr(_lib.load(), name)(ctypes.byref(args), None)
    return rc, _lib.last_error()


ADDRESS = 1 << 20                                  # stands for device memory; nothing is launched


def _cache(**kw):
    from mpsa import serving
    c = serving._Cache(ADDRESS, ADDRESS, ADDRESS, ADDRESS, 4, 64, 2, 128, 0)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


BAD_CACHES = [dict(k=None), dict(v_scale=None), dict(k=ADDRESS + 8), dict(num_pages=0), dict(page_size=48), dict(page_size=8), dict(page_size=2048), dict(Hkv=0),
              dict(D=96), dict(elem=3), dict(elem=-1), dict(num_pages=-1)]


def _norm_rope():
    from mpsa import serving
    a = serving._NormRopeArgs()
    a.x[0] = a.y[0] = ADDRESS
    a.x_sb[0] = a.x_sh[0] = a.x_sl[0] = a.y_sb[0] = a.y_sh[0] = a.y_sl[0] = 128
    a.H[0], a.B, a.L, a.D, a.norm, a.axes, a.eps = 1, 1, 1, 128, 1, 1, 1e-6
    a.cos = a.sin = ADDRESS
    a.rot, a.table_rows = 128, 10
    return a


def _set(a, name, value):
    if isinstance(value, tuple):
        getattr(a, name)[value[0]] = value[1]
    else:
        setattr(a, name, value)


@pytest.mark.parametrize("change", [dict(x=(0, None)), dict(y=(0, None)), dict(x=(1, ADDRESS)), dict(x=(0, ADDRESS + 2)), dict(in_dtype=3), dict(D=96), dict(B=0),
                                    dict(L=-1), dict(H=(0, 0)), dict(norm=3), dict(eps=-1.0), dict(eps=float("nan")), dict(x_sl=(0, 130)), dict(weight=(0, ADDRESS), w_dtype=(0, 5)),
                                    dict(weight=(0, ADDRESS), w_dtype=(0, 1)), dict(weight=(0, ADDRESS + 8)),
                                    dict(sin=None), dict(rot=0), dict(rot=12), dict(rot=136), dict(table_rows=0), dict(cos=ADDRESS + 4), dict(axes=0),
                                    dict(axes=2), dict(axes=5), dict(B=70000, L=70000)], ids=str)
def test_norm_rope_refuses(change):
    a = _norm_rope()
    for n, v in change.items():
        _set(a, n, v)
    rc, msg = _call("mpsa_norm_rope", a)
    assert rc in (-1, -2) and "norm_rope" in msg


def test_norm_rope_refuses_sections_and_long_rows():
    a = _norm_rope()
    a.axes, a.positions = 3, ADDRESS
    for ends in ((10, 5, 64), (10, 20, 63), (10, 20, 65)):
        for i, e in enumerate(ends):
            a.section_end[i] = e
        assert _call("mpsa_norm_rope", a)[0] == -1
    a = _norm_rope()
    a.norm, a.H[0] = 2, 129
    assert _call("mpsa_norm_rope", a)[0] == -2


def _append():
    from mpsa import serving
    return serving._AppendArgs(_cache(), ADDRESS, ADDRESS, 128, 128, 128, 128, 128, 128, 4, ADDRESS, ADDRESS, None, 0, 1, 1, 4)


def _read():
    from mpsa import serving
    return serving._ReadArgs(_cache(), ADDRESS, ADDRESS, 4, ADDRESS, ADDRESS, 0, 1, 1, 4)


def _attention():
    from mpsa import serving
    return serving._AttentionArgs(_cache(), ADDRESS, ADDRESS, None, ADDRESS, 1 << 40, *([128] * 6), 4, 0, ADDRESS, ADDRESS, None, None, ADDRESS, 0, 1, 1, 4, 4, 0.1)


@pytest.mark.parametrize("make,name", [(_append, "mpsa_kv_append"), (_read, "mpsa_kv_read"), (_attention, "mpsa_kv_attention")])
@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(make, name, change):
    a = make()
    a.cache = _cache(**change)
    rc, msg = _call(name, a)
    assert rc in (-1, -2) and name[5:] in msg


@pytest.mark.parametrize("make,name,change", [
    (_append, "mpsa_kv_append", dict(k=None)), (_append, "mpsa_kv_append", dict(start=None)), (_append, "mpsa_kv_append", dict(page_table=None)),
    (_append, "mpsa_kv_append", dict(in_dtype=3)), (_append, "mpsa_kv_append", dict(T=0)), (_append, "mpsa_kv_append", dict(B=70000)),
    (_append, "mpsa_kv_append", dict(max_pages=0)), (_append, "mpsa_kv_append", dict(k_sl=132)), (_append, "mpsa_kv_append", dict(v=ADDRESS + 4)),
    (_read, "mpsa_kv_read", dict(k_out=None)), (_read, "mpsa_kv_read", dict(lengths=None)), (_read, "mpsa_kv_read", dict(out_dtype=3)),
    (_read, "mpsa_kv_read", dict(max_len=0)), (_read, "mpsa_kv_read", dict(v_out=ADDRESS + 8)), (_read, "mpsa_kv_read", dict(B=70000)),
    (_attention, "mpsa_kv_attention", dict(q=None)), (_attention, "mpsa_kv_attention", dict(out=None)), (_attention, "mpsa_kv_attention", dict(lengths=None)),
    (_attention, "mpsa_kv_attention", dict(dtype=2)), (_attention, "mpsa_kv_attention", dict(T=0)), (_attention, "mpsa_kv_attention", dict(T=1025)),
    (_attention, "mpsa_kv_attention", dict(Hq=3)), (_attention, "mpsa_kv_attention", dict(Hq=0)), (_attention, "mpsa_kv_attention", dict(B=70000)),
    (_attention, "mpsa_kv_attention", dict(sm_scale=0.0)), (_attention, "mpsa_kv_attention", dict(sm_scale=float("inf"))),
    (_attention, "mpsa_kv_attention", dict(sm_scale=float("nan"))), (_attention, "mpsa_kv_attention", dict(q_sl=4)),
    (_attention, "mpsa_kv_attention", dict(out=ADDRESS + 2)), (_attention, "mpsa_kv_attention", dict(max_pages=-1)), (_attention, "mpsa_kv_attention", dict(status=None)),
    (_attention, "mpsa_kv_attention", dict(B=65535, max_pages=1 << 30)),
], ids=lambda v: str(v) if isinstance(v, dict) else None)
def test_bad_arguments_are_refused(make, name, change):
    a = make()
    for n, v in change.items():
        setattr(a, n, v)
    rc, msg = _call(name, a)
    assert rc in (-1, -2) and name[5:] in msg


def test_null_argument_blocks_are_refused():
    from mpsa import _lib
    lib = _lib.load()
    for name in ("mpsa_norm_rope", "mpsa_kv_append", "mpsa_kv_read", "mpsa_kv_attention"):
        assert getattr(lib, name)(None, None) == -1
    assert lib.mpsa_kv_attention_workspace(None) == -1


def test_argument_blocks_have_the_compilers_layout(tmp_path):
    """The ctypes structures against sizeof and the last field's offset as a C compiler sees include/mpsa.h."""
    import os
    import shutil
    import subprocess

    from mpsa import serving
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    which = [("mpsa_norm_rope_args", serving._NormRopeArgs), ("mpsa_kv_cache", serving._Cache), ("mpsa_kv_append_args", serving._AppendArgs),
             ("mpsa_kv_read_args", serving._ReadArgs), ("mpsa_kv_attention_args", serving._AttentionArgs)]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"mpsa.h\"\nint main(void) {\n"
    for name, s in which:
        src += "".join(f'printf("%zu ", offsetof({name}, {f[0]}));\n' for f in s._fields_) + f'printf("%zu\\n", sizeof({name}));\n'
    (tmp_path / "s.c").write_text(src + "return 0; }\n")
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    lines = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines()
    for (name, s), line in zip(which, lines):
        assert [int(x) for x in line.split()] == [getattr(s, f[0]).offset for f in s._fields_] + [ctypes.sizeof(s)], name


def test_host_tensors_are_refused():
    import mpsa
    x = torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    u = torch.zeros(2, 2, 16, 128, dtype=torch.uint8)
    with pytest.raises(ValueError):
        mpsa.norm_rope(x, x)
    with pytest.raises(ValueError):
        mpsa.KVCache(u, u[..., :4].contiguous(), u, u[..., :4].contiguous())
    with pytest.raises(ValueError):
        mpsa.kv_cache(2, 2, 128, device="cpu")


@pytest.mark.parametrize("elem", ["e4m3", "e5m2", "e2m1"])
def test_the_plain_rounding_is_the_nearest_value(elem):
    """The tests' own form of the cache's rounding, against a search through all values of the element type."""
    import os
    import sys
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    import serving_plain as P
    g = torch.Generator().manual_seed(0)
    x = torch.randn(60, 64, generator=g).double() * torch.exp2(torch.randint(-20, 20, (60, 1), generator=g).double())
    y, e = P.quantise(x, elem)
    t = P.element_table(elem)
    t = t[torch.isfinite(t)].unique()
    b = torch.ldexp(x.reshape(60, 2, 32), (127 - e).unsqueeze(-1))
    assert bool((b.abs().amax(-1) <= P.LARGEST[elem]).all()) and bool((b.abs().amax(-1) > P.LARGEST[elem] / 2).all())
    best = (b.unsqueeze(-1) - t).abs().amin(-1)
    assert torch.equal((b - y).abs(), best)


def test_grid_positions():
    from mpsa.model_hooks import grid_positions
    p = grid_positions((2, 3, 4), 30)
    assert p.shape == (30, 3) and p.dtype == torch.int32
    assert p[:24].tolist() == [[f, h, w] for f in range(2) for h in range(3) for w in range(4)] and int(p[24:].abs().sum()) == 0
    with pytest.raises(ValueError):
        grid_positions((2, 3, 4), 23)
