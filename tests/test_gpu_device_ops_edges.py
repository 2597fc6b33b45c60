"""Operators on caller-owned device buffers where one request's values, a value's range or several
reports at once could reach what they must not: against the definitions in 64 bits, with the
tolerances of test_gpu_device_ops.py."""
import pytest
from test_gpu_device_ops import H16, close, cross_args, cross_ref, gen, i32, kb, lora_args, lora_case, lora_ref, randn, starts_of, stream, torch_

pytestmark = pytest.mark.gpu


# every kernel choice of the projection: (lens, ids, adapters, K, N, R)
LORA_CHOICES = [
    ([1] * 24, [0, 1, -1, 2, 1, 0] * 4, 3, 256, 200, 16),                          # one launch, h beside the product
    ([1, 3, 0, 2, 5, 1] * 4, [0, 1, 2, -1, 2, 1] * 4, 3, 1024, 264, 40),            # up to 128 rows
    ([2, 1] * 90, [(i * 7) % 41 - 1 for i in range(180)], 40, 256, 264, 16),        # a few hundred of many adapters
    ([37, 90, 1, 0, 130, 64], [0, 1, -1, 2, 1, 2], 3, 256, 328, 24),                # tiles of the tensor cores
    ([1, 2] * 450, [(i * 7) % 6 - 1 for i in range(900)], 5, 128, 264, 8),          # the same, scattered rows
]


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("lens,ids,na,K,N,R", LORA_CHOICES)
def test_lora_infinities_of_an_adapter_stay_in_its_rows(lens, ids, na, K, N, R, value):
    """An adapter that rows of the call use holds infinities or NaN in some outputs' rows of B, another one
    in A: the rows of other adapters, and rows without one, are as by the definition."""
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(K + N, lens, K, N, R, na, pad=8)
    want, tol = lora_ref(x[:, :K], w, bias, a, b, scales, st, ids)
    b[1, ::7] = value
    a[2, R - 1, 3] = value
    out = torch.full((x.shape[0], N), 7.0, dtype=torch.float16, device="cuda")
    kb().lora_matmul_f16(lora_args(x, w, bias, a, b, scales, i32(st), i32(ids), out), stream())
    kb().operator_status(stream())
    row_id = torch.tensor([ad for n, ad in zip(lens, ids) for _ in range(n)], device="cuda")
    hit = torch.zeros(st[-1], N, dtype=torch.bool, device="cuda")
    hit[(row_id == 1), ::7] = True
    hit[row_id == 2] = True
    assert hit.any() and not hit.all()
    got = out[:st[-1]]
    assert not got[hit].isfinite().any()
    keep = ~hit
    close(got[keep], want[:st[-1]][keep], tol[:st[-1]][keep])


@pytest.mark.parametrize("lens,ids,na,K,N,R", LORA_CHOICES)
def test_lora_rank_product_beyond_f16(lens, ids, na, K, N, R):
    """A large scale with a small B: s x A^T passes 65,504 in some rows of an adapter, the output does not."""
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(K + R, lens, K, N, R, na, pad=8)
    scales[1] = 2.0 ** 16
    b[1] = (b[1].float() * 2.0 ** -12).half()
    if na > 3:
        scales[3], b[3] = -2.0 ** 20, (b[3].float() * 2.0 ** -16).half()
    h = x[:st[-1], :K].double() @ a[1].double().T * scales[1]
    assert (h.abs() > 65504).any() and (h.abs() < 65504).any()
    want, tol = lora_ref(x[:, :K], w, bias, a, b, scales, st, ids)
    assert want[:st[-1]].abs().max() < 60000
    out = torch.full((x.shape[0], N + 8), 7.0, dtype=torch.float16, device="cuda")
    kb().lora_matmul_f16(lora_args(x, w, bias, a, b, scales, i32(st), i32(ids), out), stream())
    kb().operator_status(stream())
    close(out[:st[-1], :N], want[:st[-1]], tol[:st[-1]])
    assert (out[st[-1]:] == 7).all() and (out[:, N:] == 7).all()


@pytest.mark.parametrize("lens,ids,na,K,N,R", LORA_CHOICES)
def test_lora_infinite_rows_stay_infinite(lens, ids, na, K, N, R):
    """A row of x with a NaN, one with an infinity, and outputs beyond f16: as by the definition."""
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(K + R, lens, K, N, R, na)
    x[0, 5], x[st[-1] - 1, K - 1] = float("nan"), float("inf")
    bias[8:16] = 65504.0
    w[9], w[12] = 0.0, 0.0
    w[9, :], w[12, 0] = w[9, :], 65504.0
    ref_x = x[:, :K].clone()
    ref_x[[0, st[-1] - 1]] = 0
    want, tol = lora_ref(ref_x, w, bias, a, b, scales, st, ids)
    out = torch.full((x.shape[0], N), 7.0, dtype=torch.float16, device="cuda")
    kb().lora_matmul_f16(lora_args(x, w, bias, a, b, scales, i32(st), i32(ids), out), stream())
    kb().operator_status(stream())
    assert out[0].isnan().all() and not out[st[-1] - 1].isfinite().any()
    mid, low = want[1:st[-1] - 1], tol[1:st[-1] - 1]
    got = out[1:st[-1] - 1]
    sure = (mid.abs() + low < 65504)  # (values next to the border may round either way)
    close(got[sure], mid[sure], low[sure])
    over = mid.abs() - low > 65520
    assert over.any() and got[over].isinf().all() and (got[over].sign() == mid[over].sign()).all()


def test_lora_starts_that_go_back_and_forth():
    """Starts that decrease again and again name 300 adapters for the two first rows: the list of a tile's
    adapters holds no more than it has room for, the report says so, and the next call is as ever."""
    torch, k = torch_(), kb()
    na, rows = 300, 2500
    x, w, bias, a, b, scales, st = lora_case(5, [rows], 1024, 64, 8, na)
    starts, ids = i32([0, 2] * (na // 2) + [rows]), i32(list(range(na)))
    out = torch.full((x.shape[0], 80), 7.0, dtype=torch.float16, device="cuda")
    k.lora_matmul_f16(lora_args(x, w, bias, a, b, scales, starts, ids, out), stream())
    with pytest.raises(k.KhError, match="starts that decrease") as e:
        k.operator_status(stream())
    assert e.value.status == 1
    assert (out[rows:] == 7).all() and (out[:, 64:] == 7).all()
    starts, ids = i32(st), i32([na - 1])
    k.lora_matmul_f16(lora_args(x, w, bias, a, b, scales, starts, ids, out), stream())
    k.operator_status(stream())
    want, tol = lora_ref(x, w, bias, a, b, scales, st, [na - 1])
    close(out[:rows, :64], want[:rows], tol[:rows])


# ---- reports ----

def bad_norm_call():
    """A norm with a position outside its table."""
    torch, k = torch_(), kb()
    x, table = randn(gen(1), 3, 64), torch.zeros(4, 128, device="cuda")
    pos = i32([0, 4, 1])
    a = k.QkNormRopeArgs(dtype=k.KH_F16, q_heads=1, head_dim=64, rotary_dim=64, eps=1e-6, rows=3, x_stride=64, out_stride=64,
                         table_rows=4, x=x.data_ptr(), out=x.data_ptr(), cossin=table.data_ptr(), positions=pos.data_ptr())
    a._keep = x, table, pos
    return a


def bad_lora_call():
    """A projection with an adapter id that does not exist."""
    torch = torch_()
    x, w, bias, a, b, scales, st = lora_case(2, [2, 2], 64, 64, 8, 2)
    starts, ids, out = i32(st), i32([0, 2]), torch.zeros(x.shape[0], 64, dtype=torch.float16, device="cuda")
    args = lora_args(x, w, bias, a, b, scales, starts, ids, out)
    args._keep = x, w, bias, a, b, scales, starts, ids, out
    return args


def test_status_reports_every_operator():
    """What two operators met before one report is in that report, and cleared by it."""
    k = kb()
    k.qk_norm_rope(bad_norm_call(), stream())
    k.lora_matmul_f16(bad_lora_call(), stream())
    with pytest.raises(k.KhError) as e:
        k.operator_status(stream())
    assert e.value.status == 1 and "position" in str(e.value) and "adapter id" in str(e.value)
    k.operator_status(stream())


def test_status_of_one_stream_keeps_to_it():
    """The report of a stream waits for that stream and finds what it met, beside work on another one."""
    torch, k = torch_(), kb()
    side = torch.cuda.Stream()
    a = bad_lora_call()
    torch.cuda.synchronize()
    busy = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for _ in range(20):
        busy.fill_(1)
    k.lora_matmul_f16(a, side.cuda_stream)
    with pytest.raises(k.KhError, match="adapter id"):
        k.operator_status(side.cuda_stream)
    k.operator_status(side.cuda_stream)
    torch.cuda.synchronize()


def test_status_of_a_capturing_stream_is_refused():
    """The report is refused before anything is done to the capture, which goes on."""
    torch, k = torch_(), kb()
    x, w, bias, a, b, scales, st = lora_case(3, [5, 6], 64, 64, 8, 2)
    starts, ids, out = i32(st), i32([0, 1]), torch.zeros(x.shape[0], 64, dtype=torch.float16, device="cuda")
    args = lora_args(x, w, bias, a, b, scales, starts, ids, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st_ = torch.cuda.current_stream().cuda_stream
        k.lora_matmul_f16(args, st_)
        with pytest.raises(k.KhError, match="captur") as e:
            k.operator_status(st_)
        assert e.value.status == 1
    graph.replay()
    torch.cuda.synchronize()
    k.operator_status(stream())
    want, tol = lora_ref(x, w, bias, a, b, scales, st, [0, 1])
    close(out[:st[-1]], want[:st[-1]], tol[:st[-1]])


def test_status_puts_waits_before_indexes_and_loses_neither():
    """A wait that gave up is reported as such, whatever was met before it, and everything is named."""
    k = kb()
    names = {"norm_index": "position", "cross_wait": "kh_cross_attention_f16: pipeline", "lora_wait": "kh_lora_matmul_f16: pipeline",
             "lora_index": "adapter id"}
    for bits in range(1, 16):
        met = [n for i, n in enumerate(names) if bits >> i & 1]
        for n in reversed(met):  # (an adapter id first, a wait of the same operator behind it)
            k.selftest_operator_status(**{n: 100 + len(n) if "wait" in n else 1}, stream=stream())
        with pytest.raises(k.KhError) as e:
            k.operator_status(stream())
        assert e.value.status == (3 if any("wait" in n for n in met) else 1), met
        for n, text in names.items():
            assert (text in str(e.value)) == (n in met)
        for n in met:
            assert "wait" not in n or f"code {100 + len(n)}" in str(e.value)
        k.operator_status(stream())


def test_status_of_a_bad_id_with_a_wait_that_gave_up():
    """The kernel's own report of an adapter id leaves room for a wait's, before and after it."""
    k = kb()
    for first in (True, False):
        if first:
            k.selftest_operator_status(lora_wait=233, stream=stream())
        k.lora_matmul_f16(bad_lora_call(), stream())
        if not first:
            k.selftest_operator_status(lora_wait=233, stream=stream())
        with pytest.raises(k.KhError, match="code 233.*adapter id") as e:
            k.operator_status(stream())
        assert e.value.status == 3
        k.operator_status(stream())


@pytest.mark.parametrize("lens", [[30, 20], [300, 0, 200], [1] * 700])
def test_lora_ids_without_adapters_are_reported(lens):
    """With no adapters at all every id is one that does not exist: none is used, and the report says so;
    the id of a segment without rows is not looked at."""
    torch, k = torch_(), kb()
    for bad in (False, True):
        x, w, bias, a, b, scales, st = lora_case(8, lens, 128, 264, 8, 1)
        starts, ids = i32(st), i32([0 if n == 0 else -1 for n in lens])
        if bad:
            ids[len(lens) - 1] = 0
        out = torch.zeros(x.shape[0], 264, dtype=torch.float16, device="cuda")
        args = lora_args(x, w, bias, a, b, scales, starts, ids, out)
        args.n_adapters, args.lora_a, args.lora_b, args.scales = 0, None, None, None
        k.lora_matmul_f16(args, stream())
        if bad:
            with pytest.raises(k.KhError, match="adapter id"):
                k.operator_status(stream())
        k.operator_status(stream())
        want, tol = lora_ref(x, w, bias, a, b, scales, st, [-1] * len(lens))
        close(out[:st[-1]], want[:st[-1]], tol[:st[-1]])


# ---- attention ----

def ones_case(top, lens_q, lens_k, D):
    """Queries of a row's constant and states of a state's constant: every score is one product."""
    torch = torch_()
    qs, ks = starts_of(lens_q), starts_of(lens_k)
    q = (top - 3.0 * torch.arange(qs[-1], device="cuda"))[:, None].expand(-1, D).half().contiguous()
    order = torch.cat([torch.randperm(n, generator=torch.Generator().manual_seed(n)) for n in lens_k]).cuda()
    k = (top - 8.0 * order)[:, None].expand(-1, D).half().contiguous()
    return q, k, randn(gen(D), ks[-1], D), qs, ks, order


@pytest.mark.parametrize("ql,kl", [([2, 16], [300, 500]), ([150, 300], [300, 500]), ([128], [700])])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_cross_scores_far_beyond_the_exponent(ql, kl, D):
    """Scores of 2^28 and more in powers of two, neighbours 2^13 and more apart (a rounding of the largest is
    2^6 at most): the output is the value of the best state, whatever the steps of f32 are up there."""
    torch = torch_()
    q, k, v, qs, ks, order = ones_case(8000.0, ql, kl, D)
    s = (q[:, :1].double() @ k[:, :1].double().T).abs() * D * 0.125 * 1.4427
    assert (s[:, order == 0] > 2.0 ** 27).all()
    out = torch.full_like(q, 7.0)
    a = cross_args(q, k, v, out, i32(qs), i32(ks), 1, 1, D, 0.125, max(ql), max(kl))
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    for i in range(len(ql)):
        best = v[ks[i] + int(order[ks[i]:ks[i + 1]].argmin())].double()
        want = best.expand(ql[i], D)
        # one state of weight 1: the exponential (2^-22), its f16 rounding and the sum's division, the output's rounding
        close(out[qs[i]:qs[i + 1]], want, (2 * H16 + 2.0 ** -20) * want.abs() + 2.0 ** -24)


@pytest.mark.parametrize("n_q", [1, 150])
@pytest.mark.parametrize("far", [16.0, 18.0, 20.0])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_cross_many_small_probabilities(n_q, far, D):
    """One state with a score 16 to 20 above 20,000 equal ones, which together still weigh 2^-9 to 2^-15: each
    of their probabilities is off by half a step of f16, relative (2^-11) or of its smallest values at the size
    in which they are kept (2^-25 where the largest is 2^7 or more: 2^-32 of it). 300 heads, so that no part of
    the states has a reference of its own."""
    torch = torch_()
    n, heads = 20_000, 300
    q = torch.ones(n_q, heads * D, dtype=torch.float16, device="cuda")
    k = torch.zeros(n, heads * D, dtype=torch.float16, device="cuda")
    k[777] = far / 8  # (exact in f16; scale 8 / D)
    head = 1 + 0.25 * randn(gen(4), n, D)
    head[777] = 0
    v = head.repeat(1, heads)
    out = torch.zeros_like(q)
    a = cross_args(q, k, v, out, i32([0, n_q]), i32([0, n]), heads, heads, D, 8.0 / D, n_q, n)
    assert a.workspace_bytes == 0
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    p = torch.softmax(k[:, :D].double().sum(1) * (8.0 / D), 0)
    size = p @ head.double().abs()
    # relative: the probabilities' and the output's rounding, and sums in f32 of n / 64 terms a part (2^-24 each,
    # twice where the tensor core cuts): 2^-14.7
    tol = (2 * H16 + 2.0 ** -14) * size + n * 2.0 ** -32 * head.double().abs().max() + 2.0 ** -25
    close(out.view(n_q, heads, D), (p @ head.double()).expand(n_q, heads, D), tol.expand(n_q, heads, D))


def test_cross_generous_bounds():
    """max_q and max_k at their limits, for buffers of a few hundred rows, with many sequences without rows:
    the CTAs are those that the buffers can need."""
    torch = torch_()
    H = KV = 12
    D, n = 64, 500
    ql, kl = [3, 140, 0, 20] + [0] * (n - 4), [70, 200, 9, 0] + [1] * (n - 4)
    qs, ks = starts_of(ql), starts_of(kl)
    q, kv = randn(gen(6), qs[-1], H * D, scale=1.5), randn(gen(7), ks[-1], 2 * KV * D)
    k, v = kv[:, :KV * D], kv[:, KV * D:]
    out = torch.full_like(q, 7.0)
    a = cross_args(q, k, v, out, i32(qs), i32(ks), H, KV, D, 0.125, 1 << 24, 1 << 24)
    assert a.workspace_bytes == 0
    kb().cross_attention_f16(a, stream())
    kb().operator_status(stream())
    want, tol = cross_ref(q, k, v, qs, ks, H, KV, D, 0.125)
    close(out, want, tol)


@pytest.mark.parametrize("G", [5, 9, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("ql,kl", [([1, 1, 1], [300, 0, 70]), ([1, 4, 90], [70, 300, 129])])
def test_cross_many_query_heads_to_a_key_head(G, ql, kl):
    """Tiles whose rows no whole number of queries fills, and single tokens on both kernels."""
    for D in (32, 64, 128):
        torch = torch_()
        KV = 2
        g = gen(G + D)
        qs, ks = starts_of(ql), starts_of(kl)
        q, kv = randn(g, qs[-1], KV * G * D, scale=1.5), randn(g, ks[-1], 2 * KV * D)
        k, v = kv[:, :KV * D], kv[:, KV * D:]
        out = torch.full((qs[-1], KV * G * D + 8), 7.0, dtype=torch.float16, device="cuda")
        a = cross_args(q, k, v, out, i32(qs), i32(ks), KV * G, KV, D, D ** -0.5, max(ql), max(kl))
        kb().cross_attention_f16(a, stream())
        kb().operator_status(stream())
        want, tol = cross_ref(q, k, v, qs, ks, KV * G, KV, D, D ** -0.5)
        close(out[:, :KV * G * D], want, tol)
        assert (out[:, KV * G * D:] == 7).all()


@pytest.mark.parametrize("max_q", [1, 30])
def test_cross_most_sequences(max_q):
    """65,535 sequences of no or one query, on no or one state: the output is the state's value."""
    torch = torch_()
    n, D = 65535, 64
    has_q = torch.rand(n, generator=gen(1), device="cuda") > 0.3
    has_k = torch.rand(n, generator=gen(2), device="cuda") > 0.3
    qs = torch.cat([torch.zeros(1, device="cuda"), has_q.cumsum(0)]).int()
    ks = torch.cat([torch.zeros(1, device="cuda"), has_k.cumsum(0)]).int()
    q, k = randn(gen(3), int(qs[-1]), D), randn(gen(4), int(ks[-1]), D)
    v = randn(gen(5), int(ks[-1]), D)
    out = torch.full_like(q, 7.0)
    b = kb()
    a = b.CrossAttentionArgs(n_seqs=n, q_heads=1, kv_heads=1, head_dim=D, max_q=max_q, max_k=1, scale=0.125, q_rows=q.shape[0],
                             kv_rows=k.shape[0], q_stride=D, k_stride=D, v_stride=D, out_stride=D, q=q.data_ptr(), k=k.data_ptr(),
                             v=v.data_ptr(), out=out.data_ptr(), q_starts=qs.data_ptr(), k_starts=ks.data_ptr())
    assert b.cross_attention_f16_workspace(a) == 0
    b.cross_attention_f16(a, stream())
    b.operator_status(stream())
    want = torch.zeros_like(q)
    both = has_q & has_k
    want[qs[:-1][both].long()] = v[ks[:-1][both].long()]
    # (a weight of one: the exponential of 2^7 and its sum, each within 2^-22)
    close(out, want.double(), H16 * want.double().abs() + 2.0 ** -25)


def test_lora_most_segments():
    """65,535 segments of no to three rows, of 60 adapters, on both sides of a tile's 128 rows."""
    torch = torch_()
    n = 65535
    lens = [(i * 7 + i // 11) % 4 for i in range(n)]
    x, w, bias, a, b, scales, st = lora_case(9, lens, 64, 72, 8, 60)
    ids = torch.tensor([(i * 13) % 61 - 1 for i in range(n)], device="cuda", dtype=torch.int32)
    out = torch.full((x.shape[0], 72), 7.0, dtype=torch.float16, device="cuda")
    starts = i32(st)
    kb().lora_matmul_f16(lora_args(x, w, bias, a, b, scales, starts, ids, out), stream())
    kb().operator_status(stream())
    row = torch.repeat_interleave(ids, torch.tensor(lens, device="cuda")).long()
    xx = x[:st[-1]].double()
    y, size = xx @ w.double().T + bias.double(), xx.abs() @ w.double().abs().T + bias.double().abs()
    tol = 64 * 2.0 ** -23 * size
    for ad in range(60):
        r = row == ad
        h, hs = xx[r] @ a[ad].double().T * scales[ad].double(), xx[r].abs() @ a[ad].double().abs().T * scales[ad].double()
        y[r] += h @ b[ad].double().T
        tol[r] += (H16 * h.abs() + 64 * 2.0 ** -23 * hs + 2.0 ** -25) @ b[ad].double().abs().T + 8 * 2.0 ** -23 * (h.abs() @ b[ad].double().abs().T)
    close(out[:st[-1]], y, tol + H16 * (y.abs() + tol) + 2.0 ** -25)
    assert (out[st[-1]:] == 7).all()


def test_streams_by_handle():
    """The legacy stream and the thread's own by their handles, and a stream of the caller's."""
    torch, k = torch_(), kb()
    for handle in (0, 1, 2, torch.cuda.Stream().cuda_stream):
        x, w, bias, a, b, scales, st = lora_case(4, [5, 6], 64, 64, 8, 2)
        starts, ids, out = i32(st), i32([0, 1]), torch.zeros(x.shape[0], 64, dtype=torch.float16, device="cuda")
        args = lora_args(x, w, bias, a, b, scales, starts, ids, out)
        torch.cuda.synchronize()
        k.lora_matmul_f16(args, handle)
        k.operator_status(handle)
        want, tol = lora_ref(x, w, bias, a, b, scales, st, [0, 1])
        close(out[:st[-1]], want[:st[-1]], tol[:st[-1]])


@pytest.mark.parametrize("D", [32, 64, 128])
def test_cross_scores_of_a_row_leave_the_others_alone(D):
    """One query with scores beyond 2^22 among others of its tile: theirs are the same bits as without it."""
    torch = torch_()
    n_q, n_k, row = 150, 700, 5
    g = gen(D)
    q, k, v = randn(g, n_q, D, scale=1.5 / 64), randn(g, n_k, D), randn(g, n_k, D)
    outs = []
    for top in (0.02, 60000.0):
        q[row] = top
        out = torch.zeros_like(q)
        a = cross_args(q, k, v, out, i32([0, n_q]), i32([0, n_k]), 1, 1, D, 8.0, n_q, n_k)
        kb().cross_attention_f16(a, stream())
        kb().operator_status(stream())
        outs.append(out)
    s = (q[row].double() @ k.double().T).abs().max() * 8 * 1.4427
    assert s > 2.0 ** 22
    others = torch.arange(n_q, device="cuda") != row
    assert torch.equal(outs[0][others], outs[1][others]) and not torch.equal(outs[0][row], outs[1][row])


@pytest.mark.parametrize("D", [32, 64, 128])
def test_cross_few_rows_leave_one_another_alone(D):
    """Up to 16 rows share a block of products: a row's bits are those that it has beside other rows."""
    torch = torch_()
    n_q, n_k = 12, 900
    g = gen(D)
    q, k, v = randn(g, n_q, D, scale=1.5), randn(g, n_k, D), randn(g, n_k, D)
    k *= torch.linspace(0.2, 3, n_k, device="cuda")[:, None].half()  # the largest scores grow along the states
    outs = []
    for size in (1.0, 0.1, 4.0):
        q2 = q * size
        q2[5] = q[5]
        out = torch.zeros_like(q)
        a = cross_args(q2, k, v, out, i32([0, n_q]), i32([0, n_k]), 1, 1, D, 0.125, n_q, n_k)
        kb().cross_attention_f16(a, stream())
        kb().operator_status(stream())
        outs.append(out[5])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
