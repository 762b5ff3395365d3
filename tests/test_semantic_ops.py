"""Refusals of the semantic head's operators and the plain forms their GPU tests compare with (CPU only)."""
import ctypes as C

import pytest
import torch

import semantic_ref as S
from fusionsense_amd import _lib, losses, ops
from fusionsense_amd.semantics import SemanticHead


def test_limits_match_the_header():
    import os
    import re
    h = open(os.path.join(os.path.dirname(_lib.__file__), "..", "include", "fsgs.h")).read()
    val = lambda n: re.search(rf"#define {n} (\S+)", h).group(1)
    assert int(val("FSGS_LINEAR_MAX_DIM")) == ops.LINEAR_MAX_DIM
    assert int(val("FSGS_DISTILL_MAX_K")) == ops.DISTILL_MAX_K
    assert int(val("FSGS_DISTILL_MAX_CLASSES")) == ops.DISTILL_MAX_CLASSES
    assert (float(val("FSGS_DISTILL_MIN_T").rstrip("f")), float(val("FSGS_DISTILL_MAX_T").rstrip("f"))) == ops.DISTILL_T_RANGE
    for name, code in ops.ACTIVATIONS.items():
        assert int(val(f"FSGS_ACT_{name.upper()}")) == code
    for name, code in ops.REDUCTIONS.items():
        assert int(val(f"FSGS_REDUCE_{name.upper()}")) == code
    for name, t in (("F32", torch.float32), ("BF16", torch.bfloat16), ("F16", torch.float16)):
        assert int(val(f"FSGS_{name}")) == ops.DTYPES[t]


def test_linear_act_refuses_what_has_no_gpu_tensor():
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_act(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(ValueError, match="float32, bfloat16"):
        ops.linear_act(torch.zeros(2, 3, dtype=torch.float64), torch.zeros(4, 3))
    with pytest.raises(ValueError, match="Tensor"):
        ops.linear_act([[1.0]], torch.zeros(1, 1))


def test_topk_distill_loss_refuses_what_has_no_gpu_tensor():
    with pytest.raises(ValueError, match="GPU"):
        losses.topk_distill_loss(torch.zeros(2, 3), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))


def test_forward_mode_tangents_go_through_autograd():
    from torch.autograd import forward_ad
    t = torch.ones(3)
    assert not ops._tracked(t, None) and ops._tracked(None, torch.ones(3, requires_grad=True))
    with torch.no_grad():
        assert not ops._tracked(torch.ones(3, requires_grad=True))
    with forward_ad.dual_level():
        d = forward_ad.make_dual(t, t)
        assert not ops._tracked(t, None) and ops._tracked(t, None, d)
        with torch.no_grad():
            assert ops._tracked(d)


# The C entries check sizes, codes and pointers before any launch: every call below returns without touching the GPU.
ONE = C.c_void_p(256)  # (never dereferenced: each of these calls is refused)


def _fwd(rows=4, k=8, n=8, dt=0, x=ONE, xp=8, w=ONE, act=0, r=None, rp=0, y=ONE):
    return _lib.load().fsgs_linear_fwd(rows, k, n, dt, x, xp, w, None, act, r, rp, y, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(k=0), dict(n=0), dict(k=65537), dict(n=65537), dict(dt=3), dict(dt=-1),
                                dict(act=4), dict(act=-1), dict(x=None), dict(w=None), dict(y=None), dict(xp=-1), dict(rp=-1),
                                dict(rows=1 << 40)])
def test_linear_fwd_entry_refuses(kw):
    assert _fwd(**kw) == -1


def test_linear_entries_without_rows_return_at_once():
    assert _fwd(rows=0, x=None, w=None, y=None) == 0
    assert _lib.load().fsgs_linear_bwd(0, 8, 8, 0, None, 8, None, None, 0, None, None, 8, None, None, None, None, 0, None) == 0


def test_linear_bwd_entry_refuses():
    lib = _lib.load()

    def bwd(rows=4, k=8, n=8, dt=0, x=ONE, act=1, dy=ONE, dyp=8, scratch=ONE, nbytes=1 << 40):
        return lib.fsgs_linear_bwd(rows, k, n, dt, x, 8, ONE, None, act, None, dy, dyp, ONE, ONE, ONE, scratch, nbytes, None)
    for kw in (dict(rows=-1), dict(k=0), dict(dt=7), dict(act=9), dict(x=None), dict(dy=None), dict(dyp=-1), dict(rows=1 << 40)):
        assert bwd(**kw) == -1, kw
    assert lib.fsgs_linear_bwd_uses_output(4, 0, 8, 0, 1) == -1
    assert lib.fsgs_linear_bwd_uses_output(4, 8, 8, 0, 1) == 0 and lib.fsgs_linear_bwd_uses_output(4, 600, 700, 1, 1) == 1
    assert lib.fsgs_linear_bwd_uses_output(4, 600, 700, 1, 2) == 0
    need = lib.fsgs_linear_bwd_scratch_bytes(4, 8, 8, 0, 1, 1, 1, 1)
    assert need > 0
    assert bwd(nbytes=need - 1) == -3 and bwd(scratch=None) == -3
    assert lib.fsgs_linear_bwd_scratch_bytes(4, 0, 8, 0, 1, 1, 1, 1) == -1


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f32", "bf16", "f16"])
def test_linear_bwd_workspace_holds_every_partial_sum(dtype, act):
    """Layers too wide for the one-pass kernel (more than 512 bytes a row, or 256 outputs): the column sums of dz take two rows
    per tile of 64 or of 128 rows, or one per 16 rows where there are 16 tiles of 128 x 128 at most; the workspace has room
    for any of them, whichever gradients come with db."""
    lib = _lib.load()
    code, e = ops.ACTIVATIONS[act], 4 if dtype == 0 else 2
    for K, N in ((64, 257), (129, 300), (200, 512), (256, 1024), (256, 4096), (300, 200), (512, 512), (768, 2050), (1024, 1500),
                 (2049, 1025), (4096, 4096), (600, 8), (513, 65536)):
        if K * e <= 512 and N <= 256:
            continue
        for rows in list(range(1, 82)) + [127, 128, 129, 1000, 2047, 2048, 2049, 2112, 5000]:
            if dtype != 0 and rows * N <= 512 and K * N <= 1 << 18:
                continue  # (one launch without a workspace)
            tiles = -(-rows // 128) * -(-N // 128)
            sums = max(2 * -(-rows // 64), 2 * -(-rows // 128), -(-rows // 16) if tiles <= 16 else 0)
            for dx, dw in ((1, 1), (0, 0), (1, 0), (0, 1)):
                room = (lib.fsgs_linear_bwd_scratch_bytes(rows, K, N, dtype, code, dx, dw, 1)
                        - lib.fsgs_linear_bwd_scratch_bytes(rows, K, N, dtype, code, dx, dw, 0))
                assert room >= 4 * N * sums, (rows, K, N, dx, dw, room, 4 * N * sums)


def _dfwd(rows=4, v=8, k=2, dt=0, s=ONE, sp=8, bits=64, idx=ONE, tdt=0, u=ONE, T=1.0, red=2, loss=ONE, scratch=ONE, nbytes=1 << 30):
    return _lib.load().fsgs_distill_fwd(rows, v, k, dt, s, sp, bits, idx, k, tdt, u, k, None, T, red, loss, None, None, scratch,
                                        nbytes, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(v=0), dict(v=524289), dict(k=0), dict(k=257), dict(dt=3), dict(tdt=3), dict(bits=16),
                                dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(T=1e-7), dict(T=2e6),
                                dict(red=3), dict(red=-1), dict(s=None), dict(idx=None), dict(u=None), dict(loss=None),
                                dict(sp=-1)])
def test_distill_fwd_entry_refuses(kw):
    assert _dfwd(**kw) == -1


def test_distill_scratch_is_checked():
    need = _lib.load().fsgs_distill_scratch_bytes()
    assert _dfwd(nbytes=need - 1) == -3 and _dfwd(scratch=None) == -3


def test_distill_bwd_entry_refuses():
    lib = _lib.load()

    def bwd(rows=4, v=8, k=2, s=ONE, stat=ONE, g=ONE, ds=ONE, T=1.0):
        return lib.fsgs_distill_bwd(rows, v, k, 0, s, v, 64, ONE, k, 0, ONE, k, None, T, stat, None, g, 0, ds, None)
    for kw in (dict(rows=-1), dict(v=0), dict(k=257), dict(s=None), dict(stat=None), dict(g=None), dict(ds=None), dict(T=0.0)):
        assert bwd(**kw) == -1, kw
    assert bwd(rows=0, s=None, stat=None, g=None, ds=None) == 0


@pytest.mark.parametrize("kw", [dict(dtype=torch.float64), dict(act="tanh"), dict(hidden=-1), dict(hidden=0, blocks=1),
                                dict(in_dim=0), dict(n_classes=0)])
def test_semantic_head_refuses(kw):
    args = dict(in_dim=4, n_classes=3)
    args.update(kw)
    with pytest.raises(ValueError):
        SemanticHead(**args)


def _coefficients(function, branch=None):
    import os
    import re
    src = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "linear.hip")).read()
    body = src[src.index(f"float {function}(") :]
    body = body[:body.index("\n}")]
    if branch is not None:
        body = body.split("} else {")[branch]
    first, rest = re.search(r"fmaf\(([-\d.e]+)f, [ta], ([-\d.e]+)f\)", body), re.findall(r"fmaf\([pq], [ta], ([-\d.e]+)f\)", body)
    scale = re.search(r"fmaf\(([\d.]+)f, fabsf", body)
    f32 = lambda v: float(torch.tensor(float(v), dtype=torch.float32))  # noqa: E731
    return [f32(v) for v in (*first.groups(), *rest)], f32(scale.group(1)) if scale else None


def test_gelu_tails_are_as_close_as_their_comments_say():
    """The normal tail's two fits, evaluated in 64 bits with the coefficients that the source holds."""
    z = torch.linspace(0, 13, 400001, dtype=torch.float64)
    e = torch.exp(-z * z / 2)
    h = 0.5 * torch.special.erfcx(z / 2 ** 0.5) * e
    c, scale = _coefficients("normal_tail")
    assert len(c) == 7
    t, p = 1 / (1 + scale * z), torch.zeros_like(z)
    for v in c:
        p = p * t + v
    assert (p * t * e - h).abs().max() < 1.3e-9
    for branch, degree in ((0, 9), (1, 7)):
        c, _ = _coefficients("normal_tail_half", branch)
        assert len(c) == degree + 1
        q = torch.zeros_like(z)
        for v in c:
            q = q * z + v
        rel = (torch.exp2(q) / h - 1).abs()
        if degree == 9:
            assert rel[z < 1].max() < 5e-6 and rel[z < 2].max() < 3.1e-5 and rel.max() < 1e-4
        else:
            assert rel[z <= 6].max() < 5.6e-6 and (z * torch.exp2(q))[z > 6].max() < 2.0 ** -26
        far, q = torch.logspace(1.2, 38, 4000, dtype=torch.float64), 0.0
        for v in c:
            q = q * far + v
        assert (q < -120).all()


def test_semantic_head_parameters():
    g = torch.Generator().manual_seed(0)
    h = SemanticHead(5, 7, hidden=6, blocks=2, generator=g)
    assert [tuple(w.shape) for w in h.weights] == [(6, 5), (6, 6), (6, 6), (7, 6)]
    assert [tuple(b.shape) for b in h.biases] == [(6,), (6,), (6,), (7,)]
    assert len(list(h.parameters())) == 8
    assert [tuple(w.shape) for w in SemanticHead(5, 7, hidden=0, blocks=0).weights] == [(7, 5)]


def test_plain_forms_agree_with_autograd():
    """The 64-bit forms' hand-written gradients against torch's, on rows of every kind."""
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*s, generator=g) for s in ((9, 5), (4, 5), (4,), (9, 4), (9, 4)))
    for kind in ops.ACTIVATIONS:
        leaves = [t.double().requires_grad_(True) for t in (x, w, b)]
        y = S.act(leaves[0] @ leaves[1].t() + leaves[2], kind) + r.double()
        want = torch.autograd.grad(y, leaves, dy.double())
        got = S.linear(x, w, b, r, kind, dy)
        assert torch.allclose(got["y"][0], y.detach(), rtol=1e-13)
        for name, t in zip(("dx", "dw", "db"), want):
            assert torch.allclose(got[name][0], t, rtol=1e-11, atol=1e-13), (kind, name)
    s = torch.randn(5, 7, generator=g).float().double().requires_grad_(True)
    idx = torch.tensor([[1, 3, -1], [2, 2, 6], [-1, 9, 7], [0, 5, 6], [4, 1, 0]])
    top = torch.randn(5, 3, generator=g)
    weight = torch.tensor([1.0, 0.5, 1.0, 0.0, 2.0])
    T = 1.7
    loss = 0.0
    for i, keep in ((0, [0, 1]), (1, [0, 1, 2]), (4, [0, 1, 2])):
        p = torch.softmax(top[i, keep].double() / T, 0)
        lq = torch.log_softmax(s[i] / T, 0)[idx[i, keep]]
        loss = loss + weight[i].double() * T * T * (p * (p.log() - lq)).sum()
    loss = loss / 3.5
    got = S.distill(s.detach().float(), idx, top, T, weight, "mean", torch.ones(()))
    grad, = torch.autograd.grad(loss, [s])
    assert abs(float(got["loss"][0]) - float(loss)) < 1e-12
    assert torch.allclose(got["dlogits"][0], grad, atol=1e-12)
