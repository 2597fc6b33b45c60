"""The operators on caller-owned device buffers against their definitions in 64 bits: per-head norm
and rotation (kh_qk_norm_rope), cross attention (kh_cross_attention_f16), projection with the
adapters of many requests (kh_lora_matmul_f16).

Tolerances count roundings. f16 rounds by at most 2^-11 of the value (2^-25 below its normal range),
f32 by 2^-24; a sum of n products in f32 is off by at most n 2^-24 of the sum of their magnitudes
(2^-23 a step where the tensor core cuts instead of rounding)."""
import math

import pytest

pytestmark = pytest.mark.gpu

H16 = 2.0 ** -11


def torch_():
    import torch
    return torch


def kb():
    from kleinhirn_b200 import backend
    return backend


def stream():
    return torch_().cuda.current_stream().cuda_stream


def gen(seed):
    return torch_().Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=None):
    torch = torch_()
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or torch.float16)


def starts_of(lens, first=0):
    s = [first]
    for n in lens:
        s.append(s[-1] + n)
    return s


def i32(v):
    return torch_().tensor(v, dtype=torch_().int32, device="cuda")


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {err[bad].max().item()} (tol {tol[bad].min().item()})"


# ---- norm and rotation ----

def norm_args(x, out, qh, kh, D, R, inter, table, pos, qw, kw, eps=1e-6):
    k = kb()
    return k.QkNormRopeArgs(
        dtype=k.KH_F16 if x.dtype == torch_().float16 else k.KH_F32, q_heads=qh, k_heads=kh, head_dim=D, rotary_dim=R,
        interleaved=int(inter), eps=eps, rows=x.shape[0], x_stride=x.stride(0), out_stride=out.stride(0),
        table_rows=0 if table is None else table.shape[0], x=x.data_ptr(), out=out.data_ptr(),
        q_weight=None if qw is None else qw.data_ptr(), k_weight=None if kw is None else kw.data_ptr(),
        cossin=None if table is None else table.data_ptr(), positions=None if pos is None else pos.data_ptr())


def norm_ref(x, qh, kh, D, R, inter, table, pos, qw, kw, eps=1e-6):
    """(y, the largest magnitude of each head's normed values), in float64."""
    torch = torch_()
    h = x[:, :(qh + kh) * D].double().view(-1, qh + kh, D)
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    if qw is not None:
        y[:, :qh] *= qw.double()
    if kw is not None:
        y[:, qh:] *= kw.double()
    top = y.abs().amax(-1, keepdim=True)
    if R:
        t = table.double()[pos.long()]
        c, s = t[:, None, :R // 2], t[:, None, R:R + R // 2]
        ia = torch.arange(0, R, 2, device="cuda") if inter else torch.arange(R // 2, device="cuda")
        ib = ia + 1 if inter else ia + R // 2
        a, b = y[..., ia], y[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y.reshape(x.shape[0], -1), top.expand_as(y).reshape(x.shape[0], -1)


def angle_table(rows, R):
    torch = torch_()
    inv = 10000.0 ** (-2.0 * torch.arange(R // 2, dtype=torch.float64, device="cuda") / max(R, 1))
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([ang.cos(), ang.cos(), ang.sin(), ang.sin()], 1).float().contiguous()


def norm_tol(x, want, top):
    """f16: one rounding of the value; f32 work: sum of squares (at most 32 steps, halved by the root),
    root, weight, angle products: below 32 roundings of the head's largest value."""
    f32 = 32 * 2.0 ** -24 * top
    return f32 + (H16 * want.abs() + 2.0 ** -25 if x.dtype == torch_().float16 else 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,qh,kh,D,R,inter,pad", [
    (1, 1, 1, 64, 64, False, 0),
    (1, 12, 0, 64, 64, False, 8),       # query heads alone
    (7, 0, 3, 32, 32, True, 0),         # key heads alone
    (33, 12, 12, 64, 64, False, 768),   # the q and k blocks of a qkv row
    (5, 8, 2, 128, 128, False, 8),
    (9, 3, 1, 128, 64, True, 0),        # half of each head rotated
    (9, 3, 1, 128, 64, False, 0),
    (4, 2, 2, 80, 80, False, 0),        # ten chunks of eight
    (4, 2, 2, 80, 40, False, 0),        # pairs 20 apart
    (4, 2, 1, 80, 40, True, 4),
    (3, 2, 1, 256, 256, False, 0),
    (3, 2, 1, 250, 34, False, 0),       # nothing aligned
    (3, 2, 1, 250, 34, True, 1),
    (6, 1, 1, 2, 2, False, 3),
    (6, 5, 1, 6, 4, True, 1),
    (6, 5, 1, 24, 0, False, 0),         # no rotation
    (1031, 5, 3, 64, 64, False, 64),
])
def test_norm_against_definition(dtype, rows, qh, kh, D, R, inter, pad):
    torch = torch_()
    dt = torch.float16 if dtype == "f16" else torch.float32
    g = gen(rows + D + R)
    x = randn(g, rows, (qh + kh) * D + pad, scale=2.0, dtype=dt)
    x[0, :D] = 0  # an all-zero head: eps alone
    table = angle_table(300, R) if R else None
    pos = torch.randint(0, 300, (rows,), generator=g, device="cuda", dtype=torch.int32) if R else None
    qw, kw = 1 + 0.3 * randn(g, D, dtype=torch.float32), None if rows == 5 else 1 + 0.3 * randn(g, D, dtype=torch.float32)
    out = torch.full((rows, (qh + kh) * D + pad), 7.0, dtype=dt, device="cuda")
    kb().qk_norm_rope(norm_args(x, out, qh, kh, D, R, inter, table, pos, qw, kw), stream())
    kb().operator_status(stream())
    want, top = norm_ref(x, qh, kh, D, R, inter, table, pos, qw, kw)
    close(out[:, :(qh + kh) * D], want, norm_tol(x, want, top))
    assert (out[:, (qh + kh) * D:] == 7).all()  # what follows the heads is left alone


def test_norm_unaligned_base_and_in_place():
    torch = torch_()
    g = gen(3)
    flat = randn(g, 40 * 300 + 1)
    x = flat[1:].view(40, 300)  # two bytes off
    table, pos = angle_table(50, 64), torch.arange(40, device="cuda", dtype=torch.int32)
    want, top = norm_ref(x, 2, 2, 64, 64, False, table, pos, None, None)
    tol = norm_tol(x, want, top)
    tail = x[:, 256:].clone()
    kb().qk_norm_rope(norm_args(x, x, 2, 2, 64, 64, False, table, pos, None, None), stream())
    close(x[:, :256], want, tol)
    assert torch.equal(x[:, 256:], tail)


def test_norm_extremes():
    """Large values stay finite (f32 squares), a NaN or infinity stays in its head."""
    torch = torch_()
    g = gen(4)
    x = randn(g, 4, 256, scale=1.0)
    x[0, :64] = 65504.0
    x[1, 64 + 3] = float("nan")
    x[2, 5] = float("inf")
    out = torch.zeros_like(x)
    kb().qk_norm_rope(norm_args(x, out, 2, 2, 64, 0, False, None, None, None, None), stream())
    assert (out[0, :64] == 1).all()
    assert out[1, 64:128].isnan().all() and out[1, :64].isfinite().all() and out[1, 128:].isfinite().all()
    assert out[2, :64].isnan().any() and out[2, 64:].isfinite().all() and out[3].isfinite().all()


def test_norm_position_outside_the_table():
    torch = torch_()
    k = kb()
    x, table = randn(gen(5), 5, 128), angle_table(10, 64)
    pos = i32([0, 10, 9, -1, 3])
    out = torch.full_like(x, 7.0)
    k.qk_norm_rope(norm_args(x, out, 1, 1, 64, 64, False, table, pos, None, None), stream())
    with pytest.raises(k.KhError, match="position"):
        k.operator_status(stream())
    k.operator_status(stream())  # reported once
    assert (out[[1, 3]] == 0).all()
    ok = [0, 2, 4]
    want, top = norm_ref(x[ok], 1, 1, 64, 64, False, table, pos[ok], None, None)
    close(out[ok], want, norm_tol(x, want, top))


# ---- cross attention ----

def cross_args(q, k, v, out, qs, ks, H, KV, D, scale, max_q, max_k, mask=None, ws=None):
    b = kb()
    a = b.CrossAttentionArgs(
        n_seqs=len(qs) - 1, q_heads=H, kv_heads=KV, head_dim=D, max_q=max_q, max_k=max_k, scale=scale, q_rows=q.shape[0],
        kv_rows=k.shape[0], q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), out_stride=out.stride(0),
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        key_mask=None if mask is None else mask.data_ptr(), q_starts=qs.data_ptr(), k_starts=ks.data_ptr())
    need = b.cross_attention_f16_workspace(a)
    a._ws = torch_().empty(max(need, 1), dtype=torch_().uint8, device="cuda") if ws is None else ws
    a._ws.fill_(0xff)  # no initial contents are needed: NaN in every type
    a.workspace, a.workspace_bytes = a._ws.data_ptr(), need
    return a


def cross_ref(q, k, v, qs, ks, H, KV, D, scale, mask=None):
    """(out, tolerance) in float64: probabilities rounded to f16 (2^-11, and 2^-25 for the small ones),
    scores off by (D + 8) 2^-23 of their magnitudes' sum, the output rounded once."""
    torch = torch_()
    out = torch.zeros(q.shape[0], H * D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    g = H // KV
    for s in range(len(qs) - 1):
        rows, st = slice(qs[s], qs[s + 1]), torch.arange(ks[s], ks[s + 1], device="cuda")
        if mask is not None:
            st = st[mask[st] > 0.5]
        if not len(st) or qs[s] == qs[s + 1]:
            continue
        for h in range(H):
            qq = q[rows, h * D:(h + 1) * D].double()
            kk, vv = (t[st, (h // g) * D:(h // g + 1) * D].double() for t in (k, v))
            p = torch.softmax(qq @ kk.T * scale, -1)
            size = abs(scale) * (qq.abs() @ kk.abs().T).amax(-1, keepdim=True)
            o, pv = p @ vv, p @ vv.abs()
            c = slice(h * D, (h + 1) * D)
            out[rows, c] = o
            # the score error moves every probability, and their sum, by its own size
            tol[rows, c] = (H16 * o.abs() + (H16 + 2 * (D + 8) * 2.0 ** -23 * (size + 1)) * pv
                            + len(st) * 2.0 ** -25 * vv.abs().max() + 2.0 ** -24)
    return out, tol


def cross_case(seed, ql, kl, H, KV, D, pad=0, first=0, scale=None):
    torch = torch_()
    g = gen(seed)
    qs, ks = starts_of(ql, first), starts_of(kl, first)
    q = randn(g, qs[-1] + 2, H * D + pad, scale=1.5)
    kv = randn(g, ks[-1] + 2, 2 * KV * D + pad)
    return q, kv, kv[:, KV * D:], qs, ks, D ** -0.5 if scale is None else scale


def cross_check(q, k, v, qs, ks, H, KV, D, scale, mask=None):
    torch = torch_()
    want, tol = cross_ref(q, k, v, qs, ks, H, KV, D, scale, mask)
    # rows of no sequence hold NaN: they must not reach a sum
    k[ks[-1]:] = float("nan")
    k[:ks[0]] = float("nan")
    out = torch.full((q.shape[0], H * D + 16), 7.0, dtype=torch.float16, device="cuda")
    mq, mk = (max([b - a for a, b in zip(s, s[1:])] + [0]) for s in (qs, ks))
    a = cross_args(q, k, v, out, i32(qs), i32(ks), H, KV, D, scale, mq, mk, mask)
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    close(out[qs[0]:qs[-1], :H * D], want[qs[0]:qs[-1]], tol[qs[0]:qs[-1]])
    assert (out[:qs[0]] == 7).all() and (out[qs[-1]:] == 7).all() and (out[:, H * D:] == 7).all()
    return out


@pytest.mark.parametrize("H,KV,D", [(2, 2, 32), (3, 3, 64), (4, 1, 64), (2, 1, 128), (6, 2, 32), (7, 1, 128)])
@pytest.mark.parametrize("ql,kl", [
    ([1], [1]),
    ([1], [129]),
    ([1, 1, 1], [5, 0, 700]),             # single tokens, one without states
    ([3, 0, 17], [64, 9, 65]),            # a sequence without queries
    ([130, 2], [127, 300]),
    ([200], [1]),
    ([70, 129, 1], [1000, 128, 257]),
])
def test_cross_against_definition(ql, kl, H, KV, D):
    q, k, v, qs, ks, scale = cross_case(H + D + len(ql), ql, kl, H, KV, D)
    cross_check(q, k, v, qs, ks, H, KV, D, scale)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("ql,kl,H,KV", [
    ([1] * 9, [2000] * 9, 4, 4),          # few rows, long states: split and joined
    ([1], [9001], 1, 1),
    ([5, 16, 4], [3001, 17, 4096], 2, 1),
    ([128], [5000], 2, 2),
    ([300], [2500], 2, 1),
    ([1] * 40, [30] * 40, 12, 12),
])
def test_cross_split_states(ql, kl, H, KV, D):
    q, k, v, qs, ks, scale = cross_case(D + len(ql), ql, kl, H, KV, D, pad=8, first=3)
    cross_check(q, k, v, qs, ks, H, KV, D, scale)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("ql,kl", [([1, 1, 1, 1], [300, 40, 513, 7]), ([140, 33, 5, 260], [300, 40, 513, 129])])
def test_cross_masks(ql, kl, D):
    """Masked states hold NaN and infinities and must not be seen; one sequence has none left (zero
    rows), one keeps only its last state, one has a whole key tile masked at its start."""
    torch = torch_()
    H, KV = 4, 2
    q, k, v, qs, ks, scale = cross_case(D, ql, kl, H, KV, D)
    mask = (torch.rand(k.shape[0], generator=gen(9), device="cuda") > 0.3).float()
    mask[ks[1]:ks[2]] = 0
    mask[ks[2]:ks[2] + 256] = 0
    mask[ks[3]:ks[4]] = 0
    mask[ks[4] - 1] = 1
    clean_k, clean_v = k.clone(), v.clone()
    off = mask <= 0.5
    k[off] = float("nan")
    v[off] = float("inf")
    want, tol = cross_ref(q, clean_k, clean_v, qs, ks, H, KV, D, scale, mask)
    out = torch.full((q.shape[0], H * D), 7.0, dtype=torch.float16, device="cuda")
    a = cross_args(q, k, v, out, i32(qs), i32(ks), H, KV, D, scale, max(ql), max(kl), mask)
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    close(out[:qs[-1]], want[:qs[-1]], tol[:qs[-1]])
    assert (out[qs[1]:qs[2]] == 0).all()


@pytest.mark.parametrize("ql,kl", [([1, 2], [400, 33]), ([150, 20], [400, 33])])
def test_cross_growing_maximum(ql, kl):
    """Scores that rise or fall along the states move the running maximum many times, or never again;
    a score range of hundreds."""
    torch = torch_()
    H, KV, D = 2, 2, 64
    for sign in (1, -1):
        q, k, v, qs, ks, _ = cross_case(11, ql, kl, H, KV, D)
        q[:, :] = q.abs()
        ramp = sign * torch.linspace(-1, 1, k.shape[0], device="cuda")[:, None]
        k[:, :KV * D] = (k[:, :KV * D].float().abs() * ramp * 3).half()
        cross_check(q, k, v, qs, ks, H, KV, D, 2.0)


def test_cross_bad_starts_stay_in_the_buffers():
    """Starts outside the buffers and decreasing ones are cut: nothing outside is read or written."""
    torch = torch_()
    H = KV = 2
    D = 64
    q, k, v, qs, ks, scale = cross_case(12, [40, 50], [300, 70], H, KV, D)
    rows = q.shape[0]
    out = torch.full((rows, H * D), 7.0, dtype=torch.float16, device="cuda")
    a = cross_args(q, k, v, out, i32([0, 40, 1 << 30]), i32([-5, 300, 1 << 30]), H, KV, D, scale, 200, 400)
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    want, tol = cross_ref(q, k, v, [0, 40, rows], [0, 300, k.shape[0]], H, KV, D, scale)
    close(out, want, tol)
    out.fill_(7)
    a = cross_args(q, k, v, out, i32([0, 40, 30]), i32([0, 300, 20]), H, KV, D, scale, 200, 400)
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    close(out[:40], want[:40], tol[:40])
    assert (out[40:] == 7).all()


def test_cross_bounds_cut_longer_sequences():
    """max_q and max_k bound what is written and read, whichever kernel takes the call."""
    torch = torch_()
    H = KV = 2
    D = 64
    for max_q in (3, 60):
        q, k, v, qs, ks, scale = cross_case(13, [100], [700], H, KV, D)
        out = torch.full((q.shape[0], H * D), 7.0, dtype=torch.float16, device="cuda")
        a = cross_args(q, k, v, out, i32(qs), i32(ks), H, KV, D, scale, max_q, 333)
        kb().cross_attention_f16(a, stream())
        kb().operator_status(stream())
        want, tol = cross_ref(q, k, v, [0, max_q], [0, 333], H, KV, D, scale)
        close(out[:max_q], want[:max_q], tol[:max_q])
        assert (out[max_q:] == 7).all()


# ---- projection with adapters ----

def lora_args(x, w, bias, a, b, scales, starts, ids, out):
    m = kb()
    args = m.LoraMatmulArgs(
        k=w.shape[1], n=w.shape[0], rank=a.shape[1], n_adapters=a.shape[0], n_segs=len(ids), rows=x.shape[0],
        x_stride=x.stride(0), out_stride=out.stride(0), x=x.data_ptr(), w=w.data_ptr(),
        bias=None if bias is None else bias.data_ptr(), lora_a=a.data_ptr(), lora_b=b.data_ptr(),
        scales=None if scales is None else scales.data_ptr(), seg_starts=starts.data_ptr(), seg_adapters=ids.data_ptr(),
        out=out.data_ptr())
    need = m.lora_matmul_f16_workspace(args)
    args._ws = torch_().empty(max(need, 1), dtype=torch_().uint8, device="cuda").fill_(0xff)
    args.workspace, args.workspace_bytes = args._ws.data_ptr(), need
    return args


def lora_ref(x, w, bias, a, b, scales, starts, ids):
    """(out, tolerance) in float64: the sums' steps, the rank product's rounding, the output's."""
    torch = torch_()
    out = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    K, R = w.shape[1], a.shape[1]
    step = 2.0 ** -23
    for i, ad in enumerate(ids):
        r = slice(starts[i], starts[i + 1])
        xx = x[r].double()
        y, size = xx @ w.double().T, xx.abs() @ w.double().abs().T
        if bias is not None:
            y, size = y + bias.double(), size + bias.double().abs()
        t = K * step * size
        if 0 <= ad < a.shape[0]:
            s = 1.0 if scales is None else scales[ad].double()
            h, hs = xx @ a[ad].double().T * s, xx.abs() @ a[ad].double().abs().T * abs(s)
            y = y + h @ b[ad].double().T
            t = t + (H16 * h.abs() + K * step * hs + 2.0 ** -25) @ b[ad].double().abs().T + R * step * (h.abs() @ b[ad].double().abs().T)
        out[r], tol[r] = y, t + H16 * (y.abs() + t) + 2.0 ** -25
    return out, tol


def lora_case(seed, lens, K, N, R, na, bias=True, scales=True, pad=0, first=0):
    torch = torch_()
    g = gen(seed)
    st = starts_of(lens, first)
    x = randn(g, st[-1] + 2, K + pad)
    x[st[-1]:] = float("nan")
    x[:st[0]] = float("nan")
    w = randn(g, N, K, scale=K ** -0.5)
    return (x, w, randn(g, N) if bias else None, randn(g, na, R, K, scale=K ** -0.5), randn(g, na, N, R, scale=R ** -0.5),
            0.5 + torch.rand(na, generator=g, device="cuda") if scales else None, st)


def lora_check(x, w, bias, a, b, scales, st, ids, out_pad=16):
    torch = torch_()
    K, N = w.shape[1], w.shape[0]
    want, tol = lora_ref(x[:, :K], w, bias, a, b, scales, st, ids)
    out = torch.full((x.shape[0], N + out_pad), 7.0, dtype=torch.float16, device="cuda")
    args = lora_args(x, w, bias, a, b, scales, i32(st), i32(ids), out)
    kb().lora_matmul_f16(args, stream())
    kb().operator_status(stream())
    close(out[st[0]:st[-1], :N], want[st[0]:st[-1]], tol[st[0]:st[-1]])
    assert (out[:st[0]] == 7).all() and (out[st[-1]:] == 7).all() and (out[:, N:] == 7).all()
    return out


@pytest.mark.parametrize("K,N,R", [(64, 64, 8), (384, 1152, 16), (768, 768, 32), (1000, 776, 24), (72, 40, 64), (520, 264, 128),
                                   (8, 8, 8)])
@pytest.mark.parametrize("lens,ids", [
    ([1], [0]),
    ([1] * 5, [2, 0, -1, 0, 2]),                        # single tokens, two requests of one adapter
    ([3, 0, 40, 100, 1, 130], [1, 0, 2, -1, 0, 1]),     # an empty request, segments across tiles
    ([700], [2]),
    ([5, 5], [-1, -1]),                                 # no adapter at all
])
def test_lora_against_definition(lens, ids, K, N, R):
    x, w, bias, a, b, scales, st = lora_case(K + N + R + len(lens), lens, K, N, R, 3, bias=len(lens) != 5, scales=len(lens) != 6,
                                             pad=8 * (len(lens) % 2), first=0 if len(lens) != 2 else 3)
    lora_check(x, w, bias, a, b, scales, st, ids)


def test_lora_many_single_rows():
    """Every row of several tiles has an adapter of its own."""
    lens = [1] * 300
    x, w, bias, a, b, scales, st = lora_case(5, lens, 256, 512, 16, 300)
    lora_check(x, w, bias, a, b, scales, st, [(i * 7) % 300 for i in range(300)])


def test_lora_large():
    lens = [37 + (i * 131) % 900 for i in range(20)]
    x, w, bias, a, b, scales, st = lora_case(6, lens, 768, 2304, 32, 5)
    lora_check(x, w, bias, a, b, scales, st, [(i % 6) - 1 for i in range(20)])


@pytest.mark.parametrize("lens", [[4, 3], [300, 200]])
def test_lora_unused_adapters_and_bad_ids(lens):
    """Adapters no request names may hold anything; an id that does not exist counts as none and is
    reported once."""
    m = kb()
    x, w, bias, a, b, scales, st = lora_case(7, lens, 128, 192, 8, 4)
    a[1], b[3] = float("nan"), float("nan")
    scales[1] = float("inf")
    lora_check(x, w, bias, a, b, scales, st, [0, 2])
    torch = torch_()
    want, tol = lora_ref(x, w, bias, a, b, scales, st, [0, -1])
    out = torch.zeros(x.shape[0], 192, dtype=torch.float16, device="cuda")
    args = lora_args(x, w, bias, a, b, scales, i32(st), i32([0, 4]), out)
    m.lora_matmul_f16(args, stream())
    with pytest.raises(m.KhError, match="adapter"):
        m.operator_status(stream())
    m.operator_status(stream())
    close(out[:st[-1]], want[:st[-1]], tol[:st[-1]])


def test_lora_without_adapters():
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(8, [30, 20], 128, 64, 8, 1)
    out = torch.zeros(x.shape[0], 64, dtype=torch.float16, device="cuda")
    args = lora_args(x, w, bias, a, b, scales, i32(st), i32([-1, -1]), out)
    args.n_adapters, args.lora_a, args.lora_b, args.scales = 0, None, None, None
    kb().lora_matmul_f16(args, stream())
    kb().operator_status(stream())
    want, tol = lora_ref(x, w, bias, a, b, scales, st, [-1, -1])
    close(out[:st[-1]], want[:st[-1]], tol[:st[-1]])


def test_lora_bad_starts_stay_in_the_buffers():
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(14, [60, 70], 128, 192, 8, 2)
    x = x[:st[-1]].contiguous()
    for starts, ids, ref in (([-9, 60, 1 << 30], [0, 1], [0, 60, 130]), ([0, 60, 50], [0, 1], [0, 50, 50])):
        out = torch.full((x.shape[0], 192), 7.0, dtype=torch.float16, device="cuda")
        kb().lora_matmul_f16(lora_args(x, w, bias, a, b, scales, i32(starts), i32(ids), out), stream())
        kb().operator_status(stream())
        want, tol = lora_ref(x, w, bias, a, b, scales, ref, ids)
        close(out[:ref[1]], want[:ref[1]], tol[:ref[1]])
        assert (out[130:] == 7).all()


# ---- streams, graphs, the run of them together ----

def test_host_memory_is_refused():
    torch, k = torch_(), kb()
    x = randn(gen(1), 4, 128)
    host = torch.zeros(4, 128, dtype=torch.float16)
    with pytest.raises(k.KhError, match="device memory"):
        k.qk_norm_rope(norm_args(x, host, 1, 1, 64, 0, False, None, None, None, None), stream())


def layer(g, lens_q, lens_k, H=4, KV=2, D=64, E=256, R=16, na=3):
    """A cross-attention layer on packed rows: adapted q and kv projections, norm and rotation of their
    heads, attention, adapted output projection. Returns (calls, outputs, inputs that may change)."""
    torch, k = torch_(), kb()
    qs, ks = starts_of(lens_q), starts_of(lens_k)
    ids = [(i * 2 + 1) % (na + 1) - 1 for i in range(len(lens_q))]
    t = {"x": randn(g, qs[-1], E), "states": randn(g, ks[-1], E), "qs": i32(qs), "ks": i32(ks), "ids": i32(ids)}
    for name, n, kk in (("q", H * D, E), ("kv", 2 * KV * D, E), ("o", E, H * D)):
        t["w" + name] = randn(g, n, kk, scale=kk ** -0.5)
        t["a" + name], t["b" + name] = randn(g, na, R, kk, scale=kk ** -0.5), randn(g, na, n, R, scale=R ** -0.5)
    t["scales"] = torch.ones(na, device="cuda")
    t["table"] = angle_table(600, D)
    t["qpos"] = torch.cat([torch.arange(n) for n in lens_q]).int().cuda()
    t["kpos"] = torch.cat([torch.arange(n) for n in lens_k]).int().cuda()
    t["qw"], t["kw"] = 1 + 0.1 * randn(g, D, dtype=torch.float32), 1 + 0.1 * randn(g, D, dtype=torch.float32)
    for name, rows, n in (("q", qs[-1], H * D), ("kv", ks[-1], 2 * KV * D), ("ctx", qs[-1], H * D), ("y", qs[-1], E)):
        t[name] = torch.zeros(rows, n, dtype=torch.float16, device="cuda")
    lq = lora_args(t["x"], t["wq"], None, t["aq"], t["bq"], t["scales"], t["qs"], t["ids"], t["q"])
    lk = lora_args(t["states"], t["wkv"], None, t["akv"], t["bkv"], t["scales"], t["ks"], t["ids"], t["kv"])
    nq = norm_args(t["q"], t["q"], H, 0, D, D, False, t["table"], t["qpos"], t["qw"], None)
    nk = norm_args(t["kv"], t["kv"], 0, KV, D, D, False, t["table"], t["kpos"], None, t["kw"])
    ca = cross_args(t["q"], t["kv"], t["kv"][:, KV * D:], t["ctx"], t["qs"], t["ks"], H, KV, D, D ** -0.5, max(lens_q), max(lens_k))
    lo = lora_args(t["ctx"], t["wo"], None, t["ao"], t["bo"], t["scales"], t["qs"], t["ids"], t["y"])

    def call(st):
        k.lora_matmul_f16(lq, st)
        k.lora_matmul_f16(lk, st)
        k.qk_norm_rope(nq, st)
        k.qk_norm_rope(nk, st)
        k.cross_attention_f16(ca, st)
        k.lora_matmul_f16(lo, st)

    t["call"], t["dims"], t["ids_host"], t["qsh"], t["ksh"] = call, (H, KV, D), ids, qs, ks
    return t


def layer_ref(t):
    """The same layer in float64 with the f16 storage of its intermediate rows."""
    torch = torch_()
    H, KV, D = t["dims"]

    def lora(x, w, a, b, st):
        return lora_ref(x, w, None, a, b, t["scales"], st, t["ids_host"])[0].half()

    q = lora(t["x"], t["wq"], t["aq"], t["bq"], t["qsh"])
    kv = lora(t["states"], t["wkv"], t["akv"], t["bkv"], t["ksh"])
    q = norm_ref(q, H, 0, D, D, False, t["table"], t["qpos"], t["qw"], None)[0].half()
    kv[:, :KV * D] = norm_ref(kv, 0, KV, D, D, False, t["table"], t["kpos"], None, t["kw"])[0].half()
    ctx = cross_ref(q, kv, kv[:, KV * D:], t["qsh"], t["ksh"], H, KV, D, D ** -0.5)[0].half()
    return lora(ctx, t["wo"], t["ao"], t["bo"], t["qsh"]).double()


def layer_close(t, want):
    # Roundings in a row: q and k (2 f16 roundings each) move a score by 4 H16 of its magnitude, at most
    # D^-1/2 |q| |k| = 8 times the weights' 1.4^2: probabilities by 2 * 4 * 16 H16 at worst and ctx with
    # them (of mean |v| about 1.2); the projections' f16 operands add one H16 each, over sums whose
    # magnitudes are about four times the output's size. 200 H16 of a typical value bounds it.
    err = (t["y"].double() - want).abs().max().item()
    assert err <= 200 * H16 * want.abs().mean().item(), (err, want.abs().mean().item())


@pytest.mark.parametrize("lens_q,lens_k", [([1] * 6, [50, 300, 7, 128, 1, 511]), ([90, 200, 3], [256, 31, 500])])
def test_layer_eager_and_replayed(lens_q, lens_k):
    torch = torch_()
    t = layer(gen(21), lens_q, lens_k)
    t["call"](stream())
    kb().operator_status(stream())
    want = layer_ref(t)
    layer_close(t, want)
    eager = t["y"].clone()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        t["call"](torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        t["y"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(t["y"], eager)  # no atomics on values: the same bits
    # other inputs in the captured buffers
    t["x"].copy_(randn(gen(22), *t["x"].shape))
    graph.replay()
    torch.cuda.synchronize()
    layer_close(t, layer_ref(t))


def test_layers_on_two_streams():
    torch = torch_()
    ts = [layer(gen(31 + i), [40 + i, 70], [300, 90]) for i in range(2)]
    torch.cuda.synchronize()
    for t in ts:
        t["call"](stream())
    torch.cuda.synchronize()
    want = [t["y"].clone() for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    for t in ts:
        t["y"].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for t, s in zip(ts, streams):
            t["call"](s.cuda_stream)
    torch.cuda.synchronize()
    for t, w in zip(ts, want):
        assert torch.equal(t["y"], w)


def test_captured_lengths_change():
    """Starts live on the device: a captured call serves other lengths within its bounds."""
    torch = torch_()
    H, KV, D = 2, 1, 64
    q, k, v, qs, ks, scale = cross_case(41, [90, 60], [500, 200], H, KV, D)
    out = torch.zeros(q.shape[0], H * D, dtype=torch.float16, device="cuda")
    dq, dk = i32(qs), i32(ks)
    a = cross_args(q, k, v, out, dq, dk, H, KV, D, scale, 100, 600)
    kb().cross_attention_f16(a, stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kb().cross_attention_f16(a, torch.cuda.current_stream().cuda_stream)
    for nq, nk in (([0, 90, 150], [0, 500, 700]), ([0, 1, 101], [0, 600, 600]), ([10, 10, 40], [100, 101, 700])):
        dq.copy_(i32(nq))
        dk.copy_(i32(nk))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = cross_ref(q, k, v, nq, nk, H, KV, D, scale)
        close(out[nq[0]:nq[-1]], want[nq[0]:nq[-1]], tol[nq[0]:nq[-1]])
        assert (out[:nq[0]] == 7).all() and (out[nq[-1]:] == 7).all()


def test_lora_adapters_scattered_over_short_segments():
    """Few adapters over many short segments: the rows of one adapter of a tile are no neighbours."""
    lens = [1 + (i * 7) % 9 for i in range(200)]
    for na in (2, 5, 40):
        x, w, bias, a, b, scales, st = lora_case(60 + na, lens, 256, 328, 24, na)
        lora_check(x, w, bias, a, b, scales, st, [(i * 5) % (na + 1) - 1 for i in range(200)])


@pytest.mark.parametrize("K,N,R", [(256, 512, 72), (72, 136, 128), (1536, 264, 8)])
def test_lora_scattered_rows_of_many_adapters(K, N, R):
    """Few rows a segment and many adapters, over several blocks of 128 rows that do not start at 0."""
    lens = [(i * 5) % 4 for i in range(200)]
    x, w, bias, a, b, scales, st = lora_case(K, lens, K, N, R, 90, pad=8, first=7)
    lora_check(x, w, bias, a, b, scales, st, [(i * 11) % 91 - 1 for i in range(200)])


@pytest.mark.parametrize("ql,kl", [([1, 3], [900, 40]), ([150, 300], [260, 90]), ([20], [4000])])
def test_cross_in_place(ql, kl):
    """out may be q, whichever kernel takes the call, with split states too."""
    H, KV, D = 4, 2, 64
    q, k, v, qs, ks, scale = cross_case(51, ql, kl, H, KV, D)
    want, tol = cross_ref(q, k, v, qs, ks, H, KV, D, scale)
    behind = q[qs[-1]:].clone()
    a = cross_args(q, k, v, q, i32(qs), i32(ks), H, KV, D, scale, max(ql), max(kl))
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    close(q[:qs[-1]], want[:qs[-1]], tol[:qs[-1]])
    assert torch_().equal(q[qs[-1]:], behind)


def test_offsets_past_32_bits():
    """Rows whose value offsets, and byte offsets, pass 2^31: the last rows of wide strided buffers."""
    torch = torch_()
    rows, width = 17000, 140000  # 2.4e9 values
    buf = torch.empty(rows, width, dtype=torch.float16, device="cuda")
    g = gen(52)
    tail = 300
    buf[-tail:, :768] = randn(g, tail, 768)
    first, qs, ks, mq, mk = rows - tail, [rows - tail, rows - 190, rows - 180], [rows - tail, rows - 90, rows], 110, 210
    H, KV, D = 4, 2, 64
    q, k, v = buf[:, :256], buf[:, 256:384], buf[:, 384:512]
    cut = [s - first for s in qs], [s - first for s in ks]
    small = [t[-tail:].clone() for t in (q, k, v)]
    want, tol = cross_ref(*small, cut[0], cut[1], H, KV, D, 0.125)
    for max_q in (mq, 4):
        out = buf[:, 512:768]
        out[-tail:] = 7
        a = cross_args(q, k, v, out, i32(qs), i32(ks), H, KV, D, 0.125, max_q, mk)
        kb().cross_attention_f16(a, stream())
        kb().operator_status(stream())
        for s in range(2):
            n = min(max_q, qs[s + 1] - qs[s])
            r = slice(cut[0][s], cut[0][s] + n)
            close(out[-tail:][r], want[r], tol[r])
            assert (out[-tail:][cut[0][s] + n:cut[0][s + 1]] == 7).all()
    w, a_, b_ = randn(g, 256, 256, scale=1 / 16), randn(g, 2, 8, 256, scale=1 / 16), randn(g, 2, 256, 8)
    for lens in ([200, 100], [2, 3]):
        st = [rows - tail, rows - tail + lens[0], rows - tail + sum(lens)]
        out = buf[:, 512:768]
        kb().lora_matmul_f16(lora_args(q, w, None, a_, b_, None, i32(st), i32([1, 0]), out), stream())
        kb().operator_status(stream())
        want, tol = lora_ref(small[0], w, None, a_, b_, None, [s - first for s in st], [1, 0])
        n = sum(lens)
        close(out[-tail:][:n], want[:n], tol[:n])
    table, pos = angle_table(rows, 64), torch.arange(rows, device="cuda").int()
    kb().qk_norm_rope(norm_args(q, q, 2, 2, 64, 64, False, table, pos, None, None), stream())
    kb().operator_status(stream())
    want, top = norm_ref(small[0], 2, 2, 64, 64, False, table, pos[-tail:], None, None)
    close(q[-tail:], want, norm_tol(small[0], want, top))


def test_two_captured_layers_replayed_at_once():
    """Two graphs with workspaces of their own, replayed on two streams at the same time."""
    torch = torch_()
    ts = [layer(gen(71 + i), [1] * 20, [300 + i] * 20) for i in range(2)] + [layer(gen(73), [60, 200], [590, 90])]
    graphs, want = [], []
    for t in ts:
        t["call"](stream())
        torch.cuda.synchronize()
        want.append(t["y"].clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            t["call"](torch.cuda.current_stream().cuda_stream)
        t["y"].zero_()
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    kb().operator_status(stream())
    for t, w in zip(ts, want):
        assert torch.equal(t["y"], w)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("D", list(range(8, 129, 8)) + [136, 176, 224, 256])
def test_norm_every_chunk_count(dtype, D):
    """Heads of 1 to 32 chunks of a load each, with the rotation over all, a part, and none of the head."""
    torch = torch_()
    g = gen(D)
    rows, qh, kh = 37, 5, 2
    x = randn(g, rows, (qh + kh) * D + 8, dtype=getattr(torch, "float16" if dtype == "f16" else "float32"))
    qw, kw = 1 + 0.1 * randn(g, D, dtype=torch.float32), 1 + 0.1 * randn(g, D, dtype=torch.float32)
    pos = torch.randint(0, 50, (rows,), generator=g, device="cuda").int()
    for R, inter in ((D, False), (D, True), (D // 16 * 8, False), (D // 16 * 8, True), (0, False)):
        table = angle_table(50, R) if R else None
        out = torch.full_like(x, 7.0)
        kb().qk_norm_rope(norm_args(x, out, qh, kh, D, R, inter, table, pos if R else None, qw, kw), stream())
        kb().operator_status(stream())
        want, top = norm_ref(x, qh, kh, D, R, inter, table, pos, qw, kw)
        close(out[:, :(qh + kh) * D], want, norm_tol(x, want, top), (R, inter))
        assert (out[:, (qh + kh) * D:] == 7).all()


@pytest.mark.parametrize("D,H,KV", [(32, 4, 4), (64, 2, 2), (64, 6, 2)])
@pytest.mark.parametrize("masked", [False, True])
def test_cross_many_queries_on_short_states(D, H, KV, masked):
    """Two row tiles to a CTA: lengths on both sides of a tile, one key tile and several, none."""
    torch = torch_()
    ql, kl = [300, 140, 1, 128, 129, 17], [256, 65, 64, 0, 1, 200]
    q, k, v, qs, ks, scale = cross_case(D + H, ql, kl, H, KV, D, pad=8, first=2)
    mask = None
    if masked:
        mask = (torch.rand(k.shape[0], generator=gen(3), device="cuda") > 0.5).float()
        mask[ks[1]:ks[2]] = 0
    out = cross_check(q, k, v, qs, ks, H, KV, D, scale, mask)
    assert (out[qs[3]:qs[4], :H * D] == 0).all()
    if masked:
        assert (out[qs[1]:qs[2], :H * D] == 0).all()


@pytest.mark.parametrize("D", [32, 64, 128])
def test_cross_join_of_many_rows(D):
    """Split states of so many rows that a warp joins each, with sequences shorter than the bounds."""
    q, k, v, qs, ks, scale = cross_case(D + 1, [400, 3, 250], [3000, 40, 1500], 3, 1, D)
    cross_check(q, k, v, qs, ks, 3, 1, D, scale)


@pytest.mark.parametrize("ql,kl", [([1, 2], [4000, 2500]), ([300, 20], [2500, 1100])])
def test_cross_split_states_captured(ql, kl):
    """Parts and their join in a graph, behind and ahead of other work on the same buffers."""
    torch = torch_()
    H, KV, D = 4, 2, 64
    q, k, v, qs, ks, scale = cross_case(81, ql, kl, H, KV, D)
    out = torch.zeros(q.shape[0], H * D, dtype=torch.float16, device="cuda")
    dq, dk = i32(qs), i32(ks)  # (the graph reads them)
    a = cross_args(q, k, v, out, dq, dk, H, KV, D, scale, max(ql), max(kl))
    assert a.workspace_bytes > 0
    kb().cross_attention_f16(a, stream())
    torch.cuda.synchronize()
    eager, twice = out.clone(), torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            a._ws.fill_(0xff)
            kb().cross_attention_f16(a, torch.cuda.current_stream().cuda_stream)
            twice.copy_(out)
            out.zero_()
    for _ in range(5):
        twice.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(twice[:qs[-1]], eager[:qs[-1]])
    kb().operator_status(stream())
    want, tol = cross_ref(q, k, v, qs, ks, H, KV, D, scale)
    close(eager[:qs[-1]], want[:qs[-1]], tol[:qs[-1]])


@pytest.mark.parametrize("lens,na", [([1] * 40, 40), ([1] * 200, 60), ([50] * 6, 3), ([1] * 5, 2)])
def test_lora_captured_back_to_back(lens, na):
    """The two launches of a projection in a graph, several projections on one workspace."""
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(82, lens, 512, 520, 16, na)
    ids = [(i * 3) % na for i in range(len(lens))]
    want, tol = lora_ref(x, w, bias, a, b, scales, st, ids)
    outs = [torch.zeros(x.shape[0], 520, dtype=torch.float16, device="cuda") for _ in range(4)]
    calls = [lora_args(x, w, bias, a, b, scales, i32(st), i32(ids), o) for o in outs]
    for c in calls:
        c._starts = i32(st), i32(ids)
        c.seg_starts, c.seg_adapters = (t.data_ptr() for t in c._starts)
        c.workspace = calls[0].workspace
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            kb().lora_matmul_f16(c, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for o in outs:
            o.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        kb().operator_status(stream())
        for o in outs:
            close(o[:st[-1]], want[:st[-1]], tol[:st[-1]])
            assert (o[st[-1]:] == 7).all()


@pytest.mark.parametrize("lens,na", [([16] * 8, 8), ([30, 1, 60, 20], 3), ([25] * 20, 16), ([40] * 24, 5)])
@pytest.mark.parametrize("K,N,R", [(1536, 136, 128), (2048, 1024, 24)])
def test_lora_adapters_of_a_tile_shared_by_clusters(lens, na, K, N, R):
    """Few row tiles of several adapters: their h is made by clusters that share the adapters."""
    x, w, bias, a, b, scales, st = lora_case(K + na, lens, K, N, R, na, first=2)
    lora_check(x, w, bias, a, b, scales, st, [(i * 3) % (na + 1) - 1 for i in range(len(lens))])
