"""The device-buffer operators around an encoder's attention, as measured calls: per-head norms of
queries and keys with the position rotation (kh_qk_norm_rope), cross attention to an encoder's packed
states (kh_cross_attention_f16) and a projection with the low-rank adapters of many requests
(kh_lora_matmul_f16).

Every case is a dict of plain values; `prepare` makes its inputs on the GPU from a seed, `run` makes
one pass (the plain torch form, or the library's call where `own` is true), `exact` the same outputs
from the definitions in 64 bits.

Definitions
- qk_norm_rope: for every row and head, y = x / sqrt(mean(x^2) + eps) * w over the head's D values (w
  one vector for the query heads, one for the key heads), then the first `rotary` values of y rotated
  by the row's position p: (a, b) -> (a cos - b sin, b cos + a sin) with angle index d for the pair
  (d, d + rotary / 2), or (2 d, 2 d + 1) in the interleaved order; cos and sin from row p of an f32
  table.
- cross_attention: sequence s has query rows [q_starts[s], q_starts[s + 1]) and state rows
  [k_starts[s], k_starts[s + 1]); query head h reads key/value head h / (q_heads / kv_heads);
  out = softmax(scale q k^T over the kept states) v, and zero where no state is kept. Rows behind the
  last sequence keep what they held.
- lora_matmul: out[t] = x[t] W^T + bias + scale[a] (x[t] A[a]^T) B[a]^T with a the adapter of the
  segment that row t lies in (-1: none). Rows behind the last segment keep what they held.
"""
import math

import torch

own = False

DEV = "cuda"
BEHIND = 3  # rows behind the last sequence of the packed buffers: an allocation is seldom exactly full


# ---- cases ----

def _norm(name, rows, q_heads, k_heads, dim, rotary, dtype="f16", interleaved=False, extra=0, table=512):
    return {"name": name, "op": "qk_norm_rope", "rows": rows, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "rotary": rotary, "dtype": dtype, "interleaved": interleaved, "extra": extra, "table": table}


def _cross(name, seqs, q_short, q_long, k_short, k_long, kv_heads, group, dim, masked=False):
    return {"name": name, "op": "cross_attention", "seqs": seqs, "q_short": q_short, "q_long": q_long,
            "k_short": k_short, "k_long": k_long, "kv_heads": kv_heads, "group": group, "dim": dim, "masked": masked}


def _lora(name, segs, short, long, k, n, adapters, rank, bias=True):
    return {"name": name, "op": "lora_matmul", "segs": segs, "short": short, "long": long, "k": k, "n": n,
            "adapters": adapters, "rank": rank, "bias": bias}


def listed():
    return [
        # one new token for each of 16 requests (12 heads of 64, the qkv row of the base encoders): latency
        _norm("norm_tokens", 16, 12, 12, 64, 64, extra=768),
        # a bulk chunk of packed base-encoder rows: the q and k blocks of 65,536 qkv rows
        _norm("norm_bulk", 65536, 12, 12, 64, 64, extra=768),
        # shared key heads of 128, half of each head rotated in neighbouring pairs, far positions, odd rows
        _norm("norm_shared", 20011, 16, 4, 128, 64, interleaved=True, extra=512, table=8192),
        # f32 activations of the small encoder (12 heads of 32)
        _norm("norm_f32", 8191, 12, 12, 32, 32, dtype="f32", extra=384),
        # one request, one query over a short text: the smallest call
        _cross("cross_one", 1, 1, 1, 128, 128, 12, 1, 32),
        # single-token step of 64 requests over their texts' states (12 heads of 64)
        _cross("cross_tokens", 64, 1, 1, 200, 512, 12, 1, 64),
        # chunks of 300-500 queries over ragged states with masked ones among them
        _cross("cross_chunks", 16, 301, 499, 700, 1500, 12, 1, 64, masked=True),
        # long prompts over long states, four query heads to a key head of 128
        _cross("cross_long", 4, 2048, 2048, 4096, 4096, 4, 4, 128),
        # one token of each of 32 requests, 8 adapters: the query projection of a step
        _lora("lora_tokens", 32, 1, 1, 768, 768, 8, 16),
        # a step of 64 requests of 48 adapters on a wide layer: weights and adapters are what is read
        _lora("lora_wide", 64, 1, 1, 4096, 4096, 48, 16, bias=False),
        # 24 ragged texts through the qkv projection of a base encoder
        _lora("lora_texts", 24, 17, 333, 768, 2304, 12, 8),
        # a bulk chunk: 256 texts of up to 510 rows, rank 32
        _lora("lora_bulk", 256, 20, 510, 768, 2304, 16, 32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "cross_attention", "lora_matmul"])
    if op == "qk_norm_rope":
        dim = rng.choice([32, 64, 64, 80, 128])
        k_heads = rng.choice([1, 2, 4, 8, 12])
        q_heads = k_heads * rng.choice([1, 1, 2, 4])
        rotary = rng.choice([dim, dim, dim // 2, 0])
        most = 65536 * 24 * 64 // ((q_heads + k_heads) * dim)
        rows = _log_int(rng, 1, min(65536, most))
        dtype = rng.choice(["f16", "f16", "f32"])
        return _nameless(_norm("", rows if dtype == "f16" else max(1, rows // 2), q_heads, k_heads, dim, rotary, dtype,
                               rng.random() < 0.4, k_heads * dim, rng.choice([512, 8192])))
    if op == "cross_attention":
        while True:
            seqs = _log_int(rng, 1, 128)
            q_long = 1 if rng.random() < 0.3 else _log_int(rng, 1, 2048)
            k_long = _log_int(rng, 1, 8192)
            kv_heads = rng.choice([1, 2, 4, 8, 12])
            group = rng.choice([1, 1, 1, 2, 3, 4, 8])
            dim = rng.choice([32, 64, 64, 128])
            scores = seqs * q_long * k_long * kv_heads * group
            states = seqs * k_long * kv_heads * dim
            if scores * dim <= 4 * 2048 * 4096 * 16 * 128 // 2 and scores <= 1 << 28 and states <= 1 << 27:
                break
        return _nameless(_cross("", seqs, max(1, int(q_long * rng.uniform(0.3, 1))), q_long,
                                max(1, int(k_long * rng.uniform(0.2, 1))), k_long, kv_heads, group, dim,
                                rng.random() < 0.4))
    while True:
        segs = _log_int(rng, 1, 256)
        long = 1 if rng.random() < 0.4 else _log_int(rng, 1, 510)
        k = rng.choice([384, 512, 768, 1000, 1024, 1152, 1536, 4096])
        n = rng.choice([384, 512, 768, 776, 1024, 1152, 1536, 2304, 4096])
        rank = rng.choice([8, 8, 16, 16, 24, 32, 64])
        if segs * long * k * n <= 68000 * 768 * 2304:
            break
    return _nameless(_lora("", segs, max(1, int(long * rng.uniform(0.1, 1))), long, k, n, rng.choice([1, 2, 5, 16, 40]),
                           rank, rng.random() < 0.5))


def _nameless(case):
    del case["name"]
    return case


def _lengths(n, short, long):
    """n lengths spread evenly over [short, long] in a mixed order, the longest among them."""
    out = [short + int((i * 0.6180339887498949) % 1.0 * (long - short + 1)) for i in range(n)]
    out[n // 2] = long
    return out


def _starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def work(case):
    if case["op"] == "qk_norm_rope":
        size = 2 if case["dtype"] == "f16" else 4
        values = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        table = min(case["rows"], case["table"]) * case["rotary"] * 4
        return {"bytes": 2 * values * size + 4 * case["rows"] + table + 8 * case["dim"],
                "flops": values * (4 + (3 if case["rotary"] else 0))}
    if case["op"] == "cross_attention":
        ql = _lengths(case["seqs"], case["q_short"], case["q_long"])
        kl = _lengths(case["seqs"], case["k_short"], case["k_long"])
        heads = case["kv_heads"] * case["group"]
        pairs = sum(a * b for a, b in zip(ql, kl))
        rows = 2 * sum(ql) * heads * case["dim"] * 2 + 2 * sum(kl) * case["kv_heads"] * case["dim"] * 2
        return {"bytes": rows + (4 * sum(kl) if case["masked"] else 0) + 8 * (case["seqs"] + 1),
                "flops": 4 * pairs * heads * case["dim"]}
    lens = _lengths(case["segs"], case["short"], case["long"])
    rows, k, n, r = sum(lens), case["k"], case["n"], case["rank"]
    ids = _adapter_ids(case)
    adapted = sum(m for m, a in zip(lens, ids) if a >= 0)
    used = len({a for a in ids if a >= 0})
    return {"bytes": 2 * (rows * (k + n) + k * n + used * r * (k + n) + (n if case["bias"] else 0)) + 8 * case["segs"],
            "flops": 2 * rows * k * n + 2 * adapted * r * (k + n)}


def _adapter_ids(case):
    """Adapter of each segment: mixed over the adapters, every eleventh segment without one."""
    return [-1 if i % 11 == 10 else (i * 7 + 3) % case["adapters"] for i in range(case["segs"])]


# ---- inputs ----

def _rand(gen, *shape, scale=1.0, dtype=torch.float16):
    return (torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "qk_norm_rope":
        dtype = torch.float16 if case["dtype"] == "f16" else torch.float32
        rows, dim, rot = case["rows"], case["dim"], case["rotary"]
        heads = case["q_heads"] + case["k_heads"]
        s["x"] = _rand(gen, rows, heads * dim + case["extra"], dtype=dtype)
        s["q_weight"] = 1 + 0.2 * _rand(gen, dim, dtype=torch.float32)
        s["k_weight"] = 1 + 0.2 * _rand(gen, dim, dtype=torch.float32)
        s["eps"] = 1e-6
        s["positions"] = torch.randint(0, case["table"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
        # cosines then sines of a row, each written for both halves (the layout of the plans' tables)
        inv = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=DEV) / max(rot, 1))
        ang = torch.arange(case["table"], dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
        s["table"] = torch.cat([ang.cos(), ang.cos(), ang.sin(), ang.sin()], dim=1).float().contiguous()
        s["out"] = torch.zeros(rows, heads * dim, dtype=dtype, device=DEV)
    elif case["op"] == "cross_attention":
        qs = _starts(_lengths(case["seqs"], case["q_short"], case["q_long"]))
        ks = _starts(_lengths(case["seqs"], case["k_short"], case["k_long"]))
        heads, kv, dim = case["kv_heads"] * case["group"], case["kv_heads"], case["dim"]
        s["q"] = _rand(gen, qs[-1] + BEHIND, heads * dim, scale=1.5)
        s["kv"] = _rand(gen, ks[-1] + BEHIND, 2 * kv * dim)  # the k and the v block of each state row
        s["mask"] = None
        if case["masked"]:
            s["mask"] = (torch.rand(ks[-1] + BEHIND, generator=gen, device=DEV) > 0.15).float()
            if case["seqs"] > 1:
                s["mask"][ks[-2]:] = 0  # the last request's states are all masked: its rows come out zero
        s["q_starts"] = torch.tensor(qs, dtype=torch.int32, device=DEV)
        s["k_starts"] = torch.tensor(ks, dtype=torch.int32, device=DEV)
        s["scale"] = dim ** -0.5
        s["out"] = torch.zeros_like(s["q"])
    else:
        starts = _starts(_lengths(case["segs"], case["short"], case["long"]))
        k, n, r, na = case["k"], case["n"], case["rank"], case["adapters"]
        s["x"] = _rand(gen, starts[-1] + BEHIND, k)
        s["w"] = _rand(gen, n, k, scale=k ** -0.5)
        s["bias"] = _rand(gen, n, scale=0.1) if case["bias"] else None
        s["a"] = _rand(gen, na, r, k, scale=k ** -0.5)
        s["b"] = _rand(gen, na, n, r, scale=0.2 * r ** -0.5)
        s["scales"] = 0.5 + 1.5 * torch.rand(na, generator=gen, device=DEV)
        s["ids_host"], s["starts_host"] = _adapter_ids(case), starts
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["ids"] = torch.tensor(s["ids_host"], dtype=torch.int32, device=DEV)
        s["out"] = torch.zeros(starts[-1] + BEHIND, n, dtype=torch.float16, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["args"] = _arguments(s)
    return s


def _arguments(s):
    """The call's arguments and workspace, which a program keeps from call to call."""
    from kleinhirn_b200 import backend
    case, out = s["case"], s["out"]
    if case["op"] == "qk_norm_rope":
        return backend.QkNormRopeArgs(
            dtype=backend.KH_F16 if case["dtype"] == "f16" else backend.KH_F32, q_heads=case["q_heads"],
            k_heads=case["k_heads"], head_dim=case["dim"], rotary_dim=case["rotary"],
            interleaved=int(case["interleaved"]), eps=s["eps"], rows=case["rows"], x_stride=s["x"].stride(0),
            out_stride=out.stride(0), table_rows=case["table"], x=s["x"].data_ptr(), out=out.data_ptr(),
            q_weight=s["q_weight"].data_ptr(), k_weight=s["k_weight"].data_ptr(), cossin=s["table"].data_ptr(),
            positions=s["positions"].data_ptr())
    if case["op"] == "cross_attention":
        a = backend.CrossAttentionArgs(
            n_seqs=case["seqs"], q_heads=case["kv_heads"] * case["group"], kv_heads=case["kv_heads"],
            head_dim=case["dim"], max_q=case["q_long"], max_k=case["k_long"], scale=s["scale"],
            q_rows=s["q"].shape[0], kv_rows=s["kv"].shape[0], q_stride=s["q"].stride(0), k_stride=s["kv"].stride(0),
            v_stride=s["kv"].stride(0), out_stride=out.stride(0), q=s["q"].data_ptr(), k=s["kv"].data_ptr(),
            v=s["kv"].data_ptr() + 2 * case["kv_heads"] * case["dim"], out=out.data_ptr(),
            key_mask=s["mask"].data_ptr() if case["masked"] else None, q_starts=s["q_starts"].data_ptr(),
            k_starts=s["k_starts"].data_ptr())
        need = backend.cross_attention_f16_workspace(a)
    else:
        a = backend.LoraMatmulArgs(
            k=case["k"], n=case["n"], rank=case["rank"], n_adapters=case["adapters"], n_segs=case["segs"],
            rows=s["x"].shape[0], x_stride=s["x"].stride(0), out_stride=out.stride(0), x=s["x"].data_ptr(),
            w=s["w"].data_ptr(), bias=s["bias"].data_ptr() if case["bias"] else None, lora_a=s["a"].data_ptr(),
            lora_b=s["b"].data_ptr(), scales=s["scales"].data_ptr(), seg_starts=s["starts"].data_ptr(),
            seg_adapters=s["ids"].data_ptr(), out=out.data_ptr())
        need = backend.lora_matmul_f16_workspace(a)
    s["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), need
    return a


# ---- one pass ----

def run(s):
    if own:
        from kleinhirn_b200 import backend
        call = {"qk_norm_rope": backend.qk_norm_rope, "cross_attention": backend.cross_attention_f16,
                "lora_matmul": backend.lora_matmul_f16}[s["case"]["op"]]
        call(s["args"], torch.cuda.current_stream().cuda_stream)
        return s["out"]
    return {"qk_norm_rope": _plain_norm, "cross_attention": _plain_cross, "lora_matmul": _plain_lora}[s["case"]["op"]](s)


def _plain_norm(s):
    c = s["case"]
    rows, qh, kh, dim, rot = c["rows"], c["q_heads"], c["k_heads"], c["dim"], c["rotary"]
    x = s["x"][:, :(qh + kh) * dim].float().view(rows, qh + kh, dim)
    w = torch.cat([s["q_weight"].expand(qh, dim), s["k_weight"].expand(kh, dim)])
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + s["eps"]) * w
    if rot:
        t = s["table"][s["positions"].long()]
        cos, sin = t[:, None, :rot // 2], t[:, None, rot:rot + rot // 2]
        if c["interleaved"]:
            p, q = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([p * cos - q * sin, q * cos + p * sin], dim=-1).flatten(-2)
        else:
            p, q = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat([p * cos - q * sin, q * cos + p * sin], dim=-1)
        y = torch.cat([turned, y[..., rot:]], dim=-1)
    return y.reshape(rows, -1).to(s["x"].dtype)


def _plain_cross(s):
    """Padded batch: every sequence at the longest one's lengths, the padding masked out."""
    c = s["case"]
    kv, g, dim = c["kv_heads"], c["group"], c["dim"]
    qi = s["q_starts"][:-1, None].long() + torch.arange(c["q_long"], device=DEV)
    ki = s["k_starts"][:-1, None].long() + torch.arange(c["k_long"], device=DEV)
    q_in, k_in = qi < s["q_starts"][1:, None], ki < s["k_starts"][1:, None]
    qi, ki = qi.clamp(max=s["q"].shape[0] - 1), ki.clamp(max=s["kv"].shape[0] - 1)
    if s["mask"] is not None:
        k_in = k_in & (s["mask"][ki] > 0.5)
    n = c["seqs"]
    q = s["q"][qi].float().view(n, c["q_long"], kv, g, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, g * c["q_long"], dim)
    kvp = s["kv"][ki].float().view(n, c["k_long"], 2, kv, dim).permute(2, 0, 3, 1, 4)
    scores = torch.matmul(q, kvp[0].transpose(-1, -2)) * s["scale"]
    keep = k_in[:, None, None, :]
    scores = scores.masked_fill(~keep, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, torch.where(k_in[:, None, :, None], kvp[1], torch.zeros_like(kvp[1])))
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.view(n, kv, g, c["q_long"], dim).permute(0, 3, 1, 2, 4).reshape(n, c["q_long"], -1)
    out = torch.zeros_like(s["q"])
    out[qi[q_in]] = o[q_in].to(out.dtype)
    return out


def _plain_lora(s):
    """All adapters' products at once, the other adapters' columns of a row cleared in between."""
    c = s["case"]
    r, na, rows = c["rank"], c["adapters"], s["starts_host"][-1]
    x = s["x"][:rows].float()
    y = x @ s["w"].float().T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    seg = torch.searchsorted(s["starts"], torch.arange(rows, device=DEV, dtype=torch.int32), right=True) - 1
    mine = s["ids"][seg][:, None] == torch.arange(na, device=DEV)
    h = (x @ s["a"].float().view(na * r, -1).T).view(rows, na, r) * (mine * s["scales"])[:, :, None]
    y = y + h.view(rows, na * r) @ s["b"].float().permute(0, 2, 1).reshape(na * r, -1)
    out = torch.zeros(s["x"].shape[0], c["n"], dtype=torch.float16, device=DEV)
    out[:rows] = y.to(torch.float16)
    return out


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "qk_norm_rope":
        dim, rot, qh = case["dim"], case["rotary"], case["q_heads"]
        out = torch.empty(case["rows"], (qh + case["k_heads"]) * dim, dtype=torch.float64, device=DEV)
        turn = s["table"].double()[s["positions"].long()]
        for h in range(qh + case["k_heads"]):
            v = s["x"][:, h * dim:(h + 1) * dim].double()
            v = v / (v.square().sum(1, keepdim=True) / dim + s["eps"]).sqrt()
            v = v * (s["q_weight"] if h < qh else s["k_weight"]).double()
            u = v.clone()
            for d in range(rot // 2):
                i, j = (2 * d, 2 * d + 1) if case["interleaved"] else (d, d + rot // 2)
                u[:, i] = v[:, i] * turn[:, d] - v[:, j] * turn[:, rot + d]
                u[:, j] = v[:, j] * turn[:, d] + v[:, i] * turn[:, rot + d]
            out[:, h * dim:(h + 1) * dim] = u
        return out
    if case["op"] == "cross_attention":
        dim, kv, g = case["dim"], case["kv_heads"], case["group"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        qs, ks = s["q_starts"].tolist(), s["k_starts"].tolist()
        for i in range(case["seqs"]):
            rows, states = slice(qs[i], qs[i + 1]), torch.arange(ks[i], ks[i + 1], device=DEV)
            if s["mask"] is not None:
                states = states[s["mask"][states] > 0.5]
            if not len(states):
                continue
            q = s["q"][rows].double().view(-1, kv, g, dim)
            k, v = s["kv"][states].double().view(-1, 2, kv, dim).unbind(1)
            for h in range(kv):
                p = torch.softmax(torch.einsum("qgd,kd->gqk", q[:, h], k[:, h]) * s["scale"], dim=-1)
                out[rows, h * g * dim:(h + 1) * g * dim] = torch.einsum("gqk,kd->qgd", p, v[:, h]).reshape(-1, g * dim)
        return out
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for i, a in enumerate(s["ids_host"]):
        rows = slice(s["starts_host"][i], s["starts_host"][i + 1])
        x = s["x"][rows].double()
        y = x @ s["w"].double().T
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if a >= 0:
            y = y + (x @ s["a"][a].double().T) @ s["b"][a].double().T * s["scales"][a].double()
        out[rows] = y
    return out
