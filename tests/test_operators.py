"""The training operators (attention, layer norm, Linear with its epilogue): refusals and the oracle's gradients on the CPU, the kernels
against the oracle in 64 bits on the GPU.  How far a result may be off comes from the oracle, element by element."""
import ctypes as C
import math
import os
import re
import sys

import pytest
import torch

from conftest import ROOT

if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
from oracle import operators_oracle as oo  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------------------------------------- CPU
def _engine_on(device):
    """An engine object without a context: what it refuses it refuses before the library is called."""
    from trafficbots_amd import hip
    from trafficbots_amd.runtime import HipEngine

    e = HipEngine.__new__(HipEngine)
    e.device, e.lib, e._ctx = torch.device(device), hip.load(), C.c_void_p()
    return e


def test_structs_of_the_operators_match_the_header():
    from trafficbots_amd import hip

    header = open(os.path.join(ROOT, "include", "trafficbots_hip.h")).read()
    for cname, cls in (("tb_attention_io", hip.TbAttentionIO), ("tb_layer_norm_io", hip.TbLayerNormIO), ("tb_linear_io", hip.TbLinearIO)):
        body = header[header.index(f"typedef struct {cname} {{"):header.index(f"}} {cname};")]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = []
        for decl in body.split("{", 1)[1].split(";"):
            for part in decl.strip().split(","):
                if part.strip():
                    names.append(re.search(r"([A-Za-z_][A-Za-z0-9_]*)\s*(\[\d+\])?$", part.strip()).group(1))
        assert names == [f[0] for f in cls._fields_], cname
    hip.load()  # (compares the sizes)
    # the packed form of a call's arguments is the ctypes one: every value a number of its own
    for cls, packer in ((hip.TbAttentionIO, hip.PACK_ATTENTION), (hip.TbLayerNormIO, hip.PACK_LAYER_NORM), (hip.TbLinearIO, hip.PACK_LINEAR)):
        assert packer.size == C.sizeof(cls)
        n, flat, io = 0, [], cls()
        for name, kind in cls._fields_:
            many = getattr(kind, "_length_", 0)
            vals = list(range(n + 1, n + 1 + max(1, many)))
            n += len(vals)
            flat += vals
            setattr(io, name, tuple(vals) if many else vals[0])
        packed = cls()
        packer.pack_into(packed, 0, *flat)
        assert bytes(packed) == bytes(io), cls


def test_workspace_sizes_refuse_what_the_operators_refuse():
    from trafficbots_amd import hip

    lib = hip.load()

    def attention(**kw):
        io = hip.TbAttentionIO()
        for k, v in dict(dict(dtype=0, n_batch=2, n_query=70, n_key=90, n_head=4, n_kv_head=2, head_dim=32), **kw).items():
            setattr(io, k, v)
        return lib.tb_attention_workspace_bytes(C.byref(io), 0), lib.tb_attention_workspace_bytes(C.byref(io), 1)

    assert attention()[0] == 0 and attention()[1] >= 4 * 2 * 4 * 70
    assert attention(n_query=20, n_key=32) == (0, 0)  # one kernel does it all
    assert attention(n_query=1, n_key=1 << 16)[0] > 0  # one query over a long cache: the walk is split
    assert attention(n_query=0) == (0, 0) and attention(n_batch=0) == (0, 0) and attention(n_key=0)[0] == 0
    for bad in (dict(dtype=2), dict(dtype=-1), dict(n_batch=-1), dict(n_query=-1), dict(n_key=-1), dict(n_head=0), dict(n_kv_head=0), dict(n_kv_head=3),
                dict(n_head=2, n_kv_head=4), dict(head_dim=7), dict(head_dim=129), dict(n_query=(1 << 30) + 1), dict(n_batch=1 << 29)):
        assert attention(**bad) == (-1, -1), bad

    def norm(**kw):
        io = hip.TbLayerNormIO()
        for k, v in dict(dict(dtype=0, n_row=5000, n_col=128), **kw).items():
            setattr(io, k, v)
        return lib.tb_layer_norm_workspace_bytes(C.byref(io), 0), lib.tb_layer_norm_workspace_bytes(C.byref(io), 1)

    assert norm()[0] == 0 and norm()[1] > 0 and norm(n_row=0) == (0, 0) and norm(n_row=40) == (0, 0)
    for bad in (dict(dtype=2), dict(n_row=-1), dict(n_col=0), dict(n_col=8193), dict(n_row=(1 << 31) + 1)):
        assert norm(**bad) == (-1, -1), bad

    def linear(**kw):
        io = hip.TbLinearIO()
        for k, v in dict(dict(dtype=1, n_row=5, n_in=11, n_out=32), **kw).items():
            setattr(io, k, v)
        return lib.tb_linear_workspace_bytes(C.byref(io), 0), lib.tb_linear_workspace_bytes(C.byref(io), 1)

    assert linear() == (0, 0) and linear(n_row=1 << 20)[1] > 0 and linear(n_in=2048)[0] > 0 and linear(n_out=2048)[1] > 0
    for bad in (dict(dtype=3), dict(n_row=-1), dict(n_in=0), dict(n_out=0), dict(activation=2), dict(n_in=(1 << 22) + 1)):
        assert linear(**bad) == (-1, -1), bad
    for f in ("tb_attention", "tb_layer_norm", "tb_linear"):
        assert getattr(lib, f + "_workspace_bytes")(None, 0) == -1
        assert getattr(lib, f)(None, None, None) != 0 and getattr(lib, f + "_backward")(None, None, None) != 0


def test_refusals_before_the_library():
    e = _engine_on("cpu")
    q, kv = torch.zeros(2, 5, 4, 8), torch.zeros(2, 6, 2, 8)
    out, lse = torch.zeros(2, 5, 4, 8), torch.zeros(2, 4, 5)
    for args, kw, what in (
        ((q[0], kv, kv), {}, "must be"),
        ((q, kv, kv[:, :5]), {}, "fit"),
        ((q, kv[:1], kv[:1]), {}, "fit"),
        ((q, kv[..., :4], kv[..., :4]), {}, "fit"),
        ((q.half(), kv.half(), kv.half()), {}, "float32 or bfloat16"),
        ((q, kv, kv.bfloat16()), {}, "one type"),
        ((q.to("meta"), kv, kv), {}, "device"),
        ((q, kv, kv), dict(key_valid=torch.ones(2, 5, dtype=torch.bool)), "key_valid"),
        ((q, kv, kv), dict(query_valid=torch.ones(2, 5)), "bool or uint8"),
        ((q, kv, kv), dict(attn_mask=torch.ones(6, 5, dtype=torch.bool)), "attn_mask"),
        ((q, kv, kv), dict(attn_mask=torch.ones(5, 6, dtype=torch.bool, device="meta")), "device"),
    ):
        with pytest.raises(ValueError, match=what):
            e.attention(*args, **kw)
        with pytest.raises(ValueError, match=what):
            e.attention_backward(out, *args, out, lse, **kw)
    for bad in ((out[:, :4], out, lse), (out, out[:, :4], lse), (out, out, lse[:, :, :4]), (out, out, lse.double()), (out.bfloat16(), out, lse)):
        with pytest.raises(ValueError):
            e.attention_backward(bad[0], q, kv, kv, bad[1], bad[2])
    x = torch.zeros(3, 8)
    w = torch.zeros(8)
    for bad in ((x.double(), w, w), (x, w[:4], w), (x, w, w.bfloat16()), (x, w, w[:4]), (torch.zeros(()), None, None)):
        with pytest.raises(ValueError):
            e.layer_norm(*bad)
    r = torch.zeros(3)
    for bad in ((x[:2], x, w, r, r), (x, x, w, r[:2], r), (x, x, w, r, r.double()), (x.bfloat16(), x, w, r, r)):
        with pytest.raises(ValueError):
            e.layer_norm_backward(*bad)
    wt = torch.zeros(4, 8)
    for kw in (dict(weight=wt[:, :5]), dict(weight=wt[0]), dict(bias=torch.zeros(3)), dict(bias=torch.zeros(4).bfloat16()), dict(activation="gelu"),
               dict(row_valid=torch.ones(4, dtype=torch.bool)), dict(row_valid=torch.ones(3)), dict(residual=torch.zeros(3, 8))):
        with pytest.raises(ValueError):
            e.linear(**dict(dict(x=x, weight=wt), **kw))
    y = torch.zeros(3, 4)
    for bad in (dict(d_out=y[:2]), dict(act=y[:, :3]), dict(act=y.bfloat16()), dict(x=x[:, :5])):
        with pytest.raises(ValueError):
            e.linear_backward(**dict(dict(d_out=y, x=x, weight=wt), **bad))


def _differences(f, x, h=1e-6):
    g = torch.zeros_like(x)
    flat, out = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        v = flat[i].item()
        flat[i] = v + h
        a = f()
        flat[i] = v - h
        out[i] = (a - f()) / (2 * h)
        flat[i] = v
    return g


def test_oracle_gradients_against_differences():
    """The formulas' gradients in the oracle are the derivatives of its forward values (central differences in 64 bits: error h^2 and
    2^-53 / h, both below 1e-8 of values around 1)."""
    g = torch.Generator().manual_seed(3)
    oo.U[torch.float64] = 2.0**-53
    try:
        q, k, v = torch.randn(2, 3, 2, 4, generator=g).double(), torch.randn(2, 5, 1, 4, generator=g).double(), torch.randn(2, 5, 1, 4, generator=g).double()
        do = torch.randn(2, 3, 2, 4, generator=g).double()
        kw = dict(query_valid=torch.tensor([[1, 1, 0], [1, 1, 1]]).bool(), key_valid=torch.tensor([[1, 0, 1, 1, 1], [0, 0, 0, 0, 0]]).bool(),
                  attn_mask=torch.rand(3, 5, generator=g) < 0.2)
        r = oo.attention(q, k, v, do, **kw)
        for name, x in (("dq", q), ("dk", k), ("dv", v)):
            d = _differences(lambda: (oo.attention(q, k, v, **kw)["out"] * do).sum().item(), x)
            assert (d - r[name]).abs().max() < 1e-7, name
        assert r["out"][1].abs().max() == 0 and (r["lse"][1] == -math.inf).all() and r["dv"][1].abs().max() == 0
        x, w, b, do = (torch.randn(*s, generator=g).double() for s in ((4, 7), (7,), (7,), (4, 7)))
        r = oo.layer_norm(x, w, b, 1e-5, do)
        for name, t in (("dx", x), ("dw", w), ("db", b)):
            d = _differences(lambda: (oo.layer_norm(x, w, b)["y"] * do).sum().item(), t)
            assert (d - r[name]).abs().max() < 1e-7, name
        x, w, b, do = (torch.randn(*s, generator=g).double() for s in ((5, 6), (3, 6), (3,), (5, 3)))
        rv = torch.tensor([1, 0, 1, 1, 1]).bool()
        r = oo.linear_backward(do, x, w, act=oo.linear(x, w, b, True, rv)["act"], row_valid=rv)
        for name, t in (("dx", x), ("dw", w), ("db", b)):
            d = _differences(lambda: (oo.linear(x, w, b, True, rv)["y"] * do).sum().item(), t)
            assert (d - r[name]).abs().max() < 1e-7, name
    finally:
        del oo.U[torch.float64]


# ------------------------------------------------------------------------------------------------- GPU
@pytest.fixture(scope="module")
def eng():
    from trafficbots_amd.config import load_model_config
    from trafficbots_amd.runtime import HipEngine

    return HipEngine(load_model_config())


def _near(what, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
    same = (got == want) | (got.isnan() & want.isnan())  # (-inf of an empty row)
    same |= want.isfinite() & (want.abs() > torch.finfo(F32).max)  # no fp32 value (dq = sum ds k ~ 1e30 * 1e15 in test_attention_values)
    bad = ~same & ~((got - want).abs() <= bound)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {got.flatten()[i]:.9g}, want {want.flatten()[i]:.9g}, "
                             f"bound {bound.flatten()[i]:.3g}")


def _attention_inputs(b, lq, lk, h, hkv, d, dtype, seed=0, pad=False, mask=None):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(b, n, hh, d, generator=g).to(dtype) for n, hh in ((lq, h), (lk, hkv), (lk, hkv), (lq, h)))
    kw = {}
    if pad:
        kw["query_valid"], kw["key_valid"] = torch.rand(b, lq, generator=g) < 0.8, torch.rand(b, lk, generator=g) < 0.7
        if b > 1:
            kw["key_valid"][0] = False  # a scene in which nothing can be seen
        for t, valid in ((q, kw["query_valid"]), (do, kw["query_valid"]), (k, kw["key_valid"]), (v, kw["key_valid"])):
            t[~valid] = float("nan")
            t[:, :, :, 0][~valid] = float("inf")
    if mask == "eye":
        kw["attn_mask"] = torch.eye(lq, lk, dtype=torch.bool)
    elif mask == "batch":
        kw["attn_mask"] = torch.rand(b, lq, lk, generator=g) < 0.5
        kw["attn_mask"][:, lq // 2] = True  # a row that sees nothing
    elif mask == "causal":
        kw["causal"] = True
    return q, k, v, do, kw


def _on(x):
    return x.cuda() if torch.is_tensor(x) else x


def _check_attention(eng, q, k, v, do, kw, ref=None):
    ref = oo.attention(q, k, v, do, **kw) if ref is None else ref
    q, k, v, do = (x.cuda() for x in (q, k, v, do))
    kw = {a: _on(x) for a, x in kw.items()}
    out, lse = eng.attention(q, k, v, **kw)
    _near("out", out, ref["out"], ref["out_bound"])
    _near("lse", lse, ref["lse"], ref["lse_bound"])
    grads = eng.attention_backward(do, q, k, v, out, lse, **kw)
    for name, x in zip(("dq", "dk", "dv"), grads):
        assert x.dtype == q.dtype
        _near(name, x, ref[name], ref[name + "_bound"])
    return (out, lse) + grads


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,lq,lk,h,hkv,d", [
    (1, 1, 1, 1, 1, 8), (2, 1, 33, 4, 4, 32), (3, 20, 20, 4, 4, 32), (2, 64, 256, 4, 4, 32), (2, 61, 61, 4, 2, 32), (1, 130, 67, 8, 2, 64),
    (2, 17, 300, 3, 1, 40), (1, 33, 31, 2, 2, 128), (1, 200, 200, 4, 1, 72), (2, 65, 129, 2, 2, 9), (3, 64, 64, 4, 2, 32), (2, 20, 31, 6, 2, 24), (2, 64, 33, 2, 1, 128), (2, 40, 64, 2, 2, 64), (1, 16, 32, 2, 1, 96), (1, 257, 15, 1, 1, 100),
])
def test_attention_sizes(eng, dtype, b, lq, lk, h, hkv, d):
    _check_attention(eng, *_attention_inputs(b, lq, lk, h, hkv, d, dtype, seed=lq + lk))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", [None, "eye", "batch", "causal"])
@pytest.mark.parametrize("pad", [False, True])
@pytest.mark.parametrize("b,lq,lk,h,hkv,d", [(3, 20, 20, 4, 4, 32), (2, 70, 70, 4, 2, 32), (2, 37, 150, 2, 1, 64), (2, 150, 37, 2, 2, 16), (2, 5, 9, 1, 1, 128)])
def test_attention_masks(eng, dtype, mask, pad, b, lq, lk, h, hkv, d):
    """Padded scenes (invalid rows hold NaN and infinity), masks that leave rows empty, causal with more queries than keys."""
    _check_attention(eng, *_attention_inputs(b, lq, lk, h, hkv, d, dtype, seed=7, pad=pad, mask=mask))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,lq,lk,h,hkv,d,mask", [(1, 1, 4097, 4, 4, 32, None), (1, 3, 2048, 8, 2, 64, "batch"), (1, 2000, 9, 4, 1, 32, None), (1, 7, 5000, 2, 1, 128, "causal"),
                                                     (2, 300, 20, 4, 2, 32, "causal"), (3, 30, 700, 2, 2, 48, "batch"), (1, 3000, 27, 2, 1, 128, None), (2, 25, 999, 4, 2, 96, None)])
def test_attention_of_few_rows_is_split_and_joined(eng, dtype, b, lq, lk, h, hkv, d, mask):
    from trafficbots_amd import hip

    io = hip.TbAttentionIO()
    io.dtype, io.n_batch, io.n_query, io.n_key, io.n_head, io.n_kv_head, io.head_dim = int(dtype == BF16), b, lq, lk, h, hkv, d
    if max(lq, lk) > 1000:
        assert eng.lib.tb_attention_workspace_bytes(C.byref(io), 1) > 4 * b * h * lq  # at least one pass is split
    _check_attention(eng, *_attention_inputs(b, lq, lk, h, hkv, d, dtype, seed=11, pad=mask is None, mask=mask))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask", [None, "batch", "causal"])
@pytest.mark.parametrize("b,lq,lk,h,hkv,d", [(5, 1, 100, 8, 1, 128), (2, 3, 70, 20, 2, 44), (1, 5, 300, 6, 1, 32), (70, 1, 66, 64, 2, 32), (3, 7, 130, 8, 2, 64), (1, 2, 2100, 32, 2, 33)])
def test_attention_of_few_rows_shares_a_walk(eng, dtype, mask, b, lq, lk, h, hkv, d):
    """The queries of all heads on one key / value head are columns of one walk: 8 to 32 of them."""
    _check_attention(eng, *_attention_inputs(b, lq, lk, h, hkv, d, dtype, seed=lq + h, pad=True, mask=mask))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_reads_and_broadcasts_views(eng, dtype):
    """One packed projection [B, L, 3, H, D], heads in front of positions, a batch-broadcast key, components that are not adjacent, masks
    that are views: the same bits as from contiguous copies."""
    g = torch.Generator().manual_seed(1)
    b, l, h, d = 2, 45, 4, 24
    packed = torch.randn(b, l, 3, h, d, generator=g).to(dtype).cuda()
    q, k, v = packed.unbind(2)
    big = torch.rand(b, 2 * l, 2 * l, generator=g).cuda() < 0.3
    for qq, kk, vv, kw in (
        (q, k, v, {}),
        (q.transpose(1, 2).contiguous().transpose(1, 2), k, v, {}),
        (q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1), {}),
        (torch.randn(b, l, d, h, generator=g).to(dtype).cuda().transpose(2, 3), k, v, {}),
        (q[:, 1::2], k, v, {}),
        (q, k, v, dict(attn_mask=big[:, :l, 3:3 + l])),
        (q, k, v, dict(attn_mask=big[:, ::2, ::2], key_valid=big[:, 0, ::2], query_valid=big[:, 1, ::2])),
        (q, k, v, dict(attn_mask=big[:1, :l, :l].expand(b, -1, -1))),
    ):
        do = torch.randn(qq.shape, generator=g).to(dtype).cuda()
        views = eng.attention(qq, kk, vv, **kw)
        views += eng.attention_backward(do.transpose(0, 1).contiguous().transpose(0, 1), qq, kk, vv, *views, **kw)
        ckw = {a: x.contiguous() for a, x in kw.items()}
        qc, kc, vc = qq.contiguous(), kk.contiguous(), vv.contiguous()
        plain = eng.attention(qc, kc, vc, **ckw)
        plain += eng.attention_backward(do, qc, kc, vc, *plain, **ckw)
        for x, y in zip(views, plain):
            assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_nothing(eng, dtype):
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)):
        q, kv, do = (torch.randn(b, n, 2, 8).to(dtype).cuda() for n in (lq, lk, lq))
        out, lse = eng.attention(q, kv, kv)
        dq, dk, dv = eng.attention_backward(do, q, kv, kv, out, lse)
        assert (out == 0).all() and (lse == -math.inf).all() and (dq == 0).all() and (dk == 0).all() and (dv == 0).all()
        assert out.shape == q.shape and dk.shape == kv.shape


@gpu
def test_attention_values(eng):
    """Scores far beyond the exponential's range, a single key, and fp32 operands over many powers of two."""
    q, k, v, do, kw = _attention_inputs(2, 40, 50, 2, 2, 32, F32, seed=2)
    _check_attention(eng, q * 30, k, v, do, kw)  # one key takes nearly all
    _check_attention(eng, q, k - 100.0, v, do, kw)  # scores around -550 and +550
    _check_attention(eng, q, k, v * 1e-20, do * 1e-12, kw)
    _check_attention(eng, q * 1e-15, k * 1e15, v * 1e20, do * 1e10, kw)
    _check_attention(eng, q, k[:, :1], v[:, :1], do, kw)
    q, k, v, do, kw = _attention_inputs(2, 40, 50, 2, 2, 32, BF16, seed=2)
    _check_attention(eng, q * 8, k, v, do, kw)
    # a NaN in a valid key reaches every query that sees it and nobody else
    k = k.clone()
    k[0, 3, 0, 5] = float("nan")
    out, lse = eng.attention(q.cuda(), k.cuda(), v.cuda())
    assert out[0, :, 0].isnan().all() and lse[0, 0].isnan().all() and not out[1].isnan().any() and not out[0, :, 1].isnan().any()


@gpu
def test_attention_offsets_beyond_32_bits(eng):
    """Keys and values whose second scene lies more than 2^31 elements behind the first."""
    g = torch.Generator().manual_seed(4)
    far = (1 << 31) + 24
    buf = torch.zeros(far + 4096, dtype=BF16, device="cuda")
    k = buf.as_strided((2, 30, 2, 16), (far, 64, 16, 1))
    v = buf.as_strided((2, 30, 2, 16), (far, 64, 16, 1), 32)
    k.copy_(torch.randn(2, 30, 2, 16, generator=g))
    v.copy_(torch.randn(2, 30, 2, 16, generator=g))
    q, do = (torch.randn(2, 9, 2, 16, generator=g).to(BF16).cuda() for _ in range(2))
    a = eng.attention(q, k, v)
    a += eng.attention_backward(do, q, k, v, *a)
    kc, vc = k.contiguous(), v.contiguous()
    c = eng.attention(q, kc, vc)
    c += eng.attention_backward(do, q, kc, vc, *c)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (5, 64), (1, 128), (300, 128), (17, 129), (70, 255), (33, 512), (9, 1000), (5, 2047), (6, 4096), (3, 8191), (2, 8192), (5000, 33), (4096, 17), (4097, 256), (600, 2000)])
def test_layer_norm(eng, dtype, rows, c):
    g = torch.Generator().manual_seed(rows + c)
    x = (torch.randn(rows, c, generator=g) * 2 + torch.randn(rows, 1, generator=g) * 5).to(dtype)
    w, b, do = torch.randn(c, generator=g).to(dtype), torch.randn(c, generator=g).to(dtype), torch.randn(rows, c, generator=g).to(dtype)
    for weight, bias in ((w, b), (None, None), (w, None)):
        ref = oo.layer_norm(x, weight, bias, 1e-5, do)
        wc, bc = (None if t is None else t.cuda() for t in (weight, bias))
        y, mean, rstd = eng.layer_norm(x.cuda(), wc, bc)
        for name, t in (("y", y), ("mean", mean), ("rstd", rstd)):
            _near(name, t, ref[name], ref[name + "_bound"])
        for name, t in zip(("dx", "dw", "db"), eng.layer_norm_backward(do.cuda(), x.cuda(), wc, mean, rstd)):
            _near(name, t, ref[name], ref[name + "_bound"])


@gpu
def test_layer_norm_shapes_and_values(eng):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 4, 5, 24, generator=g).cuda()
    y, mean, rstd = eng.layer_norm(x.transpose(0, 1), eps=1e-3)
    y2, m2, r2 = eng.layer_norm(x.transpose(0, 1).contiguous().view(-1, 24), eps=1e-3)
    assert y.shape == (4, 3, 5, 24) and mean.shape == (4, 3, 5) and torch.equal(y.reshape(-1, 24), y2) and torch.equal(rstd.flatten(), r2)
    dx, dw, db = eng.layer_norm_backward(y, x.transpose(0, 1), None, mean, rstd, want_dweight=False)
    assert dw is None and db is None and dx.shape == y.shape
    dx2, dw, db = eng.layer_norm_backward(y, x.transpose(0, 1), None, mean, rstd, want_dx=False)
    assert dx2 is None and dw.shape == (24,)
    # a constant row: y = bias; a large offset does not cost the small differences behind it
    b = torch.randn(24, generator=g).cuda()
    y, mean, rstd = eng.layer_norm(torch.full((2, 24), 3.0).cuda(), None, b)
    assert torch.equal(y, b.expand(2, -1))
    far = (torch.randn(4, 1000, generator=g) + 1e4).float()
    ref = oo.layer_norm(far)
    _near("y", eng.layer_norm(far.cuda())[0], ref["y"], ref["y_bound"])
    for rows in (0,):
        e = torch.zeros(rows, 24).cuda()
        y, mean, rstd = eng.layer_norm(e, None, b)
        dx, dw, db = eng.layer_norm_backward(e, e, None, mean, rstd)
        assert y.shape == (0, 24) and dx.shape == (0, 24) and (dw == 0).all() and (db == 0).all()
    with pytest.raises(RuntimeError, match="n_col"):
        eng.layer_norm(torch.zeros(1, 8193).cuda())
    with pytest.raises(RuntimeError, match="eps"):
        eng.layer_norm(x, eps=-1.0)


LINEAR = [(1, 1, 1), (1, 128, 128), (5, 11, 32), (70, 31, 32), (33, 128, 384), (200, 128, 128), (129, 129, 65), (16, 2048, 40), (3, 40, 1030), (14, 56, 1818), (200, 3000, 70), (1, 1100, 1), (1000, 96, 100), (257, 5, 7)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", LINEAR)
@pytest.mark.parametrize("relu,residual,pad", [(False, False, False), (True, False, True), (True, True, True), (False, True, False)])
def test_linear(eng, dtype, m, k, n, relu, residual, pad):
    g = torch.Generator().manual_seed(m + k + n)
    x, w, b, res, do = (torch.randn(*s, generator=g).to(dtype) for s in ((m, k), (n, k), (n,), (m, n), (m, n)))
    rv = torch.rand(m, generator=g) < 0.7 if pad else None
    if pad:
        x[~rv] = float("nan")
        do[~rv] = float("inf")
    ref = oo.linear(x, w, b, relu, rv, res if residual else None)
    rvc = None if rv is None else rv.cuda()
    y, act = eng.linear(x.cuda(), w.cuda(), b.cuda(), activation="relu" if relu else None, row_valid=rvc, residual=res.cuda() if residual else None, want_act=True)
    _near("y", y, ref["y"], ref["y_bound"])
    _near("act", act, ref["act"], ref["act_bound"])
    gate = act if relu else None
    ref = oo.linear_backward(do, x, w, None if gate is None else gate.cpu(), rv)
    for name, t in zip(("dx", "dw", "db"), eng.linear_backward(do.cuda(), x.cuda(), w.cuda(), act=gate, row_valid=rvc)):
        _near(name, t, ref[name], ref[name + "_bound"])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n,relu,pad", [(16384, 128, 128, True, True), (20000, 100, 37, True, False), (16500, 8, 125, False, True), (70001, 40, 8, False, False)])
def test_linear_backward_of_narrow_layers(eng, dtype, m, k, n, relu, pad):
    """Both gradient products in one walk over the rows; each alone takes the other kernels."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w, do, act = (torch.randn(*s, generator=g).to(dtype) for s in ((m, k), (n, k), (m, n), (m, n)))
    act, rv = act.clamp_min(0) if relu else None, torch.rand(m, generator=g) < 0.7 if pad else None
    if pad:
        x[~rv] = float("nan")
        do[~rv] = float("inf")
    ref = oo.linear_backward(do, x, w, act, rv)
    args = (do.cuda(), x.cuda(), w.cuda())
    kw = dict(act=_on(act), row_valid=_on(rv))
    for want in ((True, True, True), (True, True, False), (False, True, True), (True, False, False), (True, False, True)):
        for name, t, have in zip(("dx", "dw", "db"), eng.linear_backward(*args, **kw, want_dx=want[0], want_dweight=want[1], want_dbias=want[2]), want):
            assert (t is not None) == have
            if have:
                _near(name, t, ref[name], ref[name + "_bound"])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(16, 2100, 3), (5, 4096, 37), (130, 1500, 9), (1, 1040, 200)])
def test_linear_of_few_rows_and_long_sums(eng, dtype, m, k, n):
    """Few tiles and a long contraction: split and joined, forward and dx, narrower and wider than 16 bytes."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w, b, res, do = (torch.randn(*s, generator=g).to(dtype) for s in ((m, k), (n, k), (n,), (m, n), (m, k)))
    rv = torch.rand(m, generator=g) < 0.7
    x[~rv] = float("nan")
    ref = oo.linear(x, w, b, True, rv, res)
    y, act = eng.linear(x.cuda(), w.cuda(), b.cuda(), activation="relu", row_valid=rv.cuda(), residual=res.cuda(), want_act=True)
    _near("y", y, ref["y"], ref["y_bound"])
    _near("act", act, ref["act"], ref["act_bound"])
    x = torch.randn(m, n, generator=g).to(dtype)  # the other way round: dx contracts over k
    wt = w.t().contiguous()
    ref = oo.linear_backward(do, x, wt)
    for name, t in zip(("dx", "dw", "db"), eng.linear_backward(do.cuda(), x.cuda(), wt.cuda())):
        _near(name, t, ref[name], ref[name + "_bound"])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(4096, 8, 8), (5001, 128, 70), (4099, 33, 128)])
def test_linear_backward_of_narrow_layers_over_fewer_rows(eng, dtype, m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    x, w, do = (torch.randn(*s, generator=g).to(dtype) for s in ((m, k), (n, k), (m, n)))
    ref = oo.linear_backward(do, x, w)
    for name, t in zip(("dx", "dw", "db"), eng.linear_backward(do.cuda(), x.cuda(), w.cuda())):
        _near(name, t, ref[name], ref[name + "_bound"])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,lq,lk,h,d", [(160, 1, 70, 4, 32), (600, 3, 66, 1, 16), (130, 9, 300, 4, 64)])
def test_attention_of_many_problems_with_few_rows(eng, dtype, b, lq, lk, h, d):
    """More problems than workgroups that would share a walk: one wave each."""
    _check_attention(eng, *_attention_inputs(b, lq, lk, h, h, d, dtype, seed=b, pad=True))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_over_many_rows(eng, dtype):
    """The long contraction of the weight's gradient is split and joined; big tiles with ragged edges."""
    g = torch.Generator().manual_seed(0)
    m, k, n = 20011, 136, 150
    x, w, do = (torch.randn(*s, generator=g).to(dtype) for s in ((m, k), (n, k), (m, n)))
    ref, back = oo.linear(x, w), oo.linear_backward(do, x, w)
    _near("y", eng.linear(x.cuda(), w.cuda()), ref["y"], ref["y_bound"])
    for name, t in zip(("dx", "dw", "db"), eng.linear_backward(do.cuda(), x.cuda(), w.cuda())):
        _near(name, t, back[name], back[name + "_bound"])


@gpu
@pytest.mark.parametrize("m,k,n,relu,residual,pad", [(16500, 64, 300, False, True, False), (16500, 128, 300, True, True, True), (33000, 192, 600, True, False, True),
                                                      (32768, 64, 512, False, False, False), (40000, 128, 510, False, True, True)])
def test_linear_with_direct_loads(eng, m, k, n, relu, residual, pad):
    """bf16 rows of whole 128-byte lines: tiles of 128 and 256, odd and even numbers of steps, ragged edges."""
    g = torch.Generator().manual_seed(m + k + n)
    x, w, b, res = (torch.randn(*s, generator=g).to(BF16) for s in ((m, k), (n, k), (n,), (m, n)))
    rv = torch.rand(m, generator=g) < 0.7 if pad else None
    if pad:
        x[~rv] = float("nan")
    ref = oo.linear(x, w, b, relu, rv, res if residual else None)
    kw = dict(activation="relu" if relu else None, row_valid=None if rv is None else rv.cuda(), residual=res.cuda() if residual else None, want_act=True)
    y, act = eng.linear(x.cuda(), w.cuda(), b.cuda(), **kw)
    _near("y", y, ref["y"], ref["y_bound"])
    _near("act", act, ref["act"], ref["act_bound"])
    # the same operands one element off the 16-byte grid take the other kernel: within the bound too
    off = torch.empty(m * k + 1, dtype=BF16, device="cuda")[1:].view(m, k)
    off.copy_(x)
    _near("y", eng.linear(off, w.cuda(), b.cuda(), **kw)[0], ref["y"], ref["y_bound"])


@gpu
def test_linear_shapes_and_wishes(eng):
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(3, 4, 20, generator=g).cuda(), torch.randn(30, 20, generator=g).cuda(), torch.randn(30, generator=g).cuda()
    y = eng.linear(x.transpose(0, 1), w, b)
    assert y.shape == (4, 3, 30) and torch.equal(y.reshape(12, 30), eng.linear(x.transpose(0, 1).reshape(12, 20), w, b))
    dx, dw, db = eng.linear_backward(y, x.transpose(0, 1), w)
    assert dx.shape == (4, 3, 20) and dw.shape == (30, 20) and db.shape == (30,)
    for want in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        r = eng.linear_backward(y, x.transpose(0, 1), w, want_dx=want[0], want_dweight=want[1], want_dbias=want[2])
        for have, t, full in zip(want, r, (dx, dw, db)):
            assert torch.equal(t, full) if have else t is None
    e = torch.zeros(0, 20).cuda()
    assert eng.linear(e, w, b).shape == (0, 30)
    dx, dw, db = eng.linear_backward(torch.zeros(0, 30).cuda(), e, w)
    assert dx.shape == (0, 20) and (dw == 0).all() and (db == 0).all()


@gpu
def test_linear_offsets_beyond_32_bits(eng):
    m, k = (1 << 25) + 5, 72
    x = torch.zeros(m, k, dtype=BF16, device="cuda")  # 2^31.2 elements
    g = torch.Generator().manual_seed(4)
    tail = torch.randn(37, k, generator=g).to(BF16).cuda()
    x[-37:] = tail
    w = torch.randn(8, k, generator=g).to(BF16).cuda()
    y = eng.linear(x, w)
    ref = oo.linear(tail.cpu(), w.cpu())
    _near("y", y[-37:], ref["y"], ref["y_bound"])
    assert (y[:-37] == 0).all()
    dx, dw, db = eng.linear_backward(y, x, w)
    ref = oo.linear_backward(y[-37:].cpu(), tail.cpu(), w.cpu())
    _near("dx", dx[-37:], ref["dx"], ref["dx_bound"])
    assert (dx[:-37] == 0).all()
    _near("dw", dw, ref["dw"], ref["dw_bound"])
    _near("db", db, ref["db"], ref["db_bound"])


def _layer(f, p, src, tgt, src_valid, tgt_valid, h):
    """The reference's pre-norm layer (transformer.py:189-239): attention of the normed source over the normed target, residual, then the
    feed-forward and its residual; rows without a visible target keep their value through the attention block, padded rows end as 0."""
    b, ls, c = src.shape
    s, t = f["norm"](src, p["n1w"], p["n1b"]), f["norm"](tgt, p["ntw"], p["ntb"])
    q = f["linear"](s, p["wq"], p["bq"]).view(b, ls, h, c // h)
    kv = f["linear"](t, p["wkv"], p["bkv"]).view(b, tgt.shape[1], 2, h, c // h)
    a = f["attention"](q, kv[:, :, 0], kv[:, :, 1], src_valid, tgt_valid).reshape(b, ls, c)
    sees = src_valid & tgt_valid.any(1, keepdim=True)
    src = f["linear"](a, p["wo"], p["bo"], row_valid=sees, residual=src)
    u = f["linear"](f["norm"](src, p["n2w"], p["n2b"]), p["w1"], p["b1"], activation="relu")
    src = f["linear"](u, p["w2"], p["b2"], residual=src)
    return src.masked_fill(~src_valid[..., None], 0)


def _plain_ops():
    def linear(x, w, b, activation=None, row_valid=None, residual=None):
        y = x @ w.t() + b
        y = y.clamp_min(0) if activation else y
        y = y if row_valid is None else y.masked_fill(~row_valid[..., None], 0)
        return y if residual is None else y + residual

    def norm(x, w, b):
        m = x.mean(-1, keepdim=True)
        return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * w + b

    def attention(q, k, v, query_valid, key_valid):
        s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(q.shape[-1])
        s = s.masked_fill(~key_valid[:, None, None], -1e30)
        p = s.softmax(-1) * key_valid[:, None, None] * query_valid[:, None, :, None]
        return torch.einsum("bhij,bjhd->bihd", p, v)

    return {"linear": linear, "norm": norm, "attention": attention}


def _layer_case(dtype):
    g = torch.Generator().manual_seed(12)
    b, ls, lt, c, h = 6, 40, 70, 128, 4
    shapes = dict(n1w=(c,), n1b=(c,), ntw=(c,), ntb=(c,), n2w=(c,), n2b=(c,), wq=(c, c), bq=(c,), wkv=(2 * c, c), bkv=(2 * c,), wo=(c, c), bo=(c,), w1=(c, c),
                  b1=(c,), w2=(c, c), b2=(c,))
    p = {k: torch.randn(*s, generator=g) * (c**-0.5 if len(s) == 2 else 0.1) + (1.0 if k in ("n1w", "ntw", "n2w") else 0.0) for k, s in shapes.items()}
    src, tgt, up = torch.randn(b, ls, c, generator=g), torch.randn(b, lt, c, generator=g), torch.randn(b, ls, c, generator=g)
    sv, tv = torch.rand(b, ls, generator=g) < 0.8, torch.rand(b, lt, generator=g) < 0.8
    tv[2] = False
    return {k: v.to(dtype) for k, v in p.items()}, src.to(dtype), tgt.to(dtype), up.to(dtype), sv, tv, h


def _functional(eng):
    from trafficbots_amd import functional as fn

    return {"linear": lambda *a, **k: fn.linear(eng, *a, **k), "norm": lambda x, w, b: fn.layer_norm(eng, x, w, b),
            "attention": lambda q, k, v, qv, kv: fn.attention(eng, q, k, v, query_valid=qv, key_valid=kv)}


@gpu
def test_transformer_layer_trains(eng):
    """One layer of the policy through the autograd forms, loss and every gradient against 64-bit autograd of the plain formulas.  fp32: the
    longest chain of products (d src through both blocks) has ~10 operators, each within a few hundred 2^-24 of its terms' size."""
    p, src, tgt, up, sv, tv, h = _layer_case(F32)

    def run(f, dtype, dev):
        leaves = {k: v.to(dev, dtype).requires_grad_() for k, v in dict(p, src=src, tgt=tgt).items()}
        y = _layer(f, leaves, leaves["src"], leaves["tgt"], sv.to(dev), tv.to(dev), h)
        y.backward(up.to(dev, dtype))
        return y, {k: v.grad for k, v in leaves.items()}

    y, grads = run(_functional(eng), F32, "cuda")
    want, want_grads = run(_plain_ops(), torch.float64, "cpu")
    for name, a, b in [("y", y, want)] + [(k, grads[k], want_grads[k]) for k in want_grads]:
        rel = ((a.double().cpu() - b).norm() / b.norm()).item()
        assert rel < 2e-5, (name, rel)
    # a second backward through the same graph's results is refused, not wrong
    x = src.cuda().requires_grad_()
    o = _functional(eng)["norm"](x, p["n1w"].cuda(), p["n1b"].cuda())
    (gx,) = torch.autograd.grad(o.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@gpu
def test_transformer_layer_forward_bf16(eng):
    """bf16: ten operators in a row, each within 2^-8 (its result) + 2^-8 (attention's probabilities) of its terms."""
    p, src, tgt, up, sv, tv, h = _layer_case(BF16)
    y = _layer(_functional(eng), {k: v.cuda() for k, v in p.items()}, src.cuda(), tgt.cuda(), sv.cuda(), tv.cuda(), h)
    want = _layer(_plain_ops(), {k: v.double() for k, v in p.items()}, src.double(), tgt.double(), sv, tv, h)
    rel = ((y.double().cpu() - want).norm() / want.norm()).item()
    assert rel < 11 * 2.0**-8, rel


def _step(eng, t):
    """Forward and backward calls of a layer's operators on fixed buffers."""
    y, mean, rstd = eng.layer_norm(t["x"], t["w"], t["b"])
    q = eng.linear(y, t["wq"], t["b"])
    z = q.view(q.shape[0], q.shape[1], 4, -1)
    out, lse = eng.attention(z, z, z, key_valid=t["kv"], query_valid=t["kv"])
    u, act = eng.linear(out.reshape(y.shape), t["wq"], t["b"], activation="relu", residual=t["x"], want_act=True)
    du, dw, db = eng.linear_backward(t["g"], out.reshape(y.shape), t["wq"], act=act)
    dq, dk, dv = eng.attention_backward(du.view(z.shape), z, z, z, out, lse, key_valid=t["kv"], query_valid=t["kv"])
    dx, dn, dm = eng.layer_norm_backward(dq.reshape(y.shape), t["x"], t["w"], mean, rstd)
    one = eng.attention(z[:1, :1], z[:1], z[:1])  # (a single row: the split path)
    return [u, dw, db, dq, dk, dv, dx, dn, dm, *one]


def _step_inputs(seed, dtype, l=2500):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(2, l, 128, generator=g), "w": torch.randn(128, generator=g), "b": torch.randn(128, generator=g) * 0.1,
         "wq": torch.randn(128, 128, generator=g) * 0.09, "g": torch.randn(2, l, 128, generator=g)}
    t = {k: v.to(dtype).cuda() for k, v in t.items()}
    t["kv"] = (torch.rand(2, l, generator=g) < 0.8).cuda()
    return t


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_operators_in_graphs_and_on_streams(eng, dtype):
    """The same bits: called twice, on a side stream, captured into two graphs that are replayed in turn with other inputs between the replays,
    beside eager calls."""
    t = _step_inputs(1, dtype)
    want = _step(eng, t)
    assert all(torch.equal(a, b) for a, b in zip(want, _step(eng, t)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _step(eng, t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    torch.cuda.synchronize()
    graphs = []
    for seed in (1, 2):
        buf = _step_inputs(seed, dtype)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = _step(eng, buf)
        graphs.append((gr, buf, res))
    for seed in (3, 4, 5):
        new = _step_inputs(seed, dtype)
        for gr, buf, res in graphs:
            for k in buf:
                buf[k].copy_(new[k])
            gr.replay()
        eager = _step(eng, new)
        for gr, buf, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(eager, res)), seed
            gr.replay()
        torch.cuda.synchronize()
        for gr, buf, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(eager, res)), seed


@gpu
def test_the_current_device_and_the_library_errors(eng):
    """A refused call leaves a message and no trace; the calling thread's device is what it was."""
    before = torch.cuda.current_device()
    q = torch.zeros(1, 2, 1, 130).cuda()
    with pytest.raises(RuntimeError, match="head_dim"):
        eng.attention(q, q, q)
    q = torch.zeros(1, 2, 3, 8).cuda()
    with pytest.raises(RuntimeError, match="multiple"):
        eng.attention(q, q[:, :, :2], q[:, :, :2])
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="scale"):
            eng.attention(q, q, q, scale=bad)
    out, lse = eng.attention(q, q, q, scale=0.5)
    assert (out == 0).all() and torch.allclose(lse, torch.full_like(lse, math.log(2)))
    assert torch.cuda.current_device() == before
    from trafficbots_amd import hip

    io = hip.TbAttentionIO()
    io.n_batch = io.n_query = io.n_key = io.n_head = io.n_kv_head = 1
    io.head_dim = 8
    io.scale = 1.0
    assert eng.lib.tb_attention(eng._ctx, C.byref(io), None) != 0 and b"NULL" in eng.lib.tb_last_error(eng._ctx)
    io.n_key, io.n_head, io.n_kv_head = 1 << 16, 1, 1
    io.q = io.k = io.v = io.out = io.lse = lse.data_ptr()
    assert eng.lib.tb_attention(eng._ctx, C.byref(io), None) != 0 and b"workspace" in eng.lib.tb_last_error(eng._ctx)


@gpu
def test_linear_gradients_need_their_operands(eng):
    """The C entry refuses what its kernels would read through a null pointer."""
    from trafficbots_amd import hip

    t = torch.zeros(4, 16).cuda()
    for fields, wish in ((("weight", "d_out"), "dbias"), (("weight", "d_out"), "dweight"), (("x", "d_out"), "dx"), (("x", "weight"), "dx"), (("x", "weight"), "dbias")):
        io = hip.TbLinearIO()
        io.n_in, io.n_out, io.n_row = 16, 16, 4
        for f in fields + (wish,):
            setattr(io, f, t.data_ptr())
        assert eng.lib.tb_linear_backward(eng._ctx, C.byref(io), None) != 0 and b"NULL" in eng.lib.tb_last_error(eng._ctx)


@gpu
def test_forms_notice_operands_that_changed_before_the_gradient(eng):
    from trafficbots_amd import functional as fn

    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 5, 2, 16, generator=g).cuda().requires_grad_()
    x, w = torch.randn(6, 16, generator=g).cuda().requires_grad_(), torch.randn(8, 16, generator=g).cuda().requires_grad_()
    kv, am, rv = torch.ones(2, 5, dtype=torch.bool).cuda(), torch.zeros(5, 5, dtype=torch.bool).cuda(), torch.ones(6, dtype=torch.bool).cuda()
    for y, mask in ((fn.attention(eng, q, q, q, key_valid=kv), kv), (fn.attention(eng, q, q, q, attn_mask=am), am), (fn.linear(eng, x, w, row_valid=rv), rv)):
        mask.logical_not_()
        with pytest.raises(RuntimeError, match="modified"):
            y.sum().backward()
    y = fn.linear(eng, x, w, activation="relu")
    y += 1  # ReLU's gradient needs it
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


@gpu
def test_calls_of_two_threads(eng):
    """Two threads on streams of their own, one context: the same bits as alone."""
    import threading

    inputs = [_step_inputs(s, F32) for s in (1, 2)]
    want = [_step(eng, t) for t in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = _step(eng, inputs[i])
            s.synchronize()
        except Exception as e:  # noqa: BLE001 (reported below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_an_engine_on_the_device_without_an_index(eng):
    from trafficbots_amd.runtime import HipEngine

    e = HipEngine(eng.cfg, "cuda")
    x = torch.randn(3, 16, generator=torch.Generator().manual_seed(0)).cuda()
    assert e.device == x.device and torch.equal(e.linear(x, x), eng.linear(x, x))
