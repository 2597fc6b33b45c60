"""Refusals of the operators on caller-owned device buffers (kh_qk_norm_rope, kh_cross_attention_f16,
kh_lora_matmul_f16): sizes, strides, alignment and pointers are judged on the host before anything is
queued, so these run without a device (the pointers are never followed)."""
import ctypes

import pytest

from kleinhirn_b200 import backend as kb

P = 1 << 20  # an aligned address that no refused call may follow


def norm(**kw):
    a = dict(dtype=kb.KH_F16, q_heads=2, k_heads=2, head_dim=64, rotary_dim=64, interleaved=0, eps=1e-6, rows=3,
             x_stride=256, out_stride=256, table_rows=8, x=P, out=2 * P, q_weight=P, k_weight=P, cossin=P, positions=P)
    a.update(kw)
    return kb.QkNormRopeArgs(**a)


def cross(**kw):
    a = dict(n_seqs=2, q_heads=4, kv_heads=2, head_dim=64, max_q=5, max_k=9, scale=0.125, q_rows=10, kv_rows=18,
             q_stride=256, k_stride=128, v_stride=128, out_stride=256, q=P, k=P, v=P, out=2 * P, key_mask=None,
             q_starts=P, k_starts=P, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    return kb.CrossAttentionArgs(**a)


def lora(**kw):
    a = dict(k=64, n=128, rank=8, n_adapters=3, n_segs=2, rows=10, x_stride=64, out_stride=128, x=P, w=P, bias=None,
             lora_a=P, lora_b=P, scales=None, seg_starts=P, seg_adapters=P, out=2 * P, workspace=P,
             workspace_bytes=1 << 40)
    a.update(kw)
    return kb.LoraMatmulArgs(**a)


def refused(call, args, text):
    with pytest.raises(kb.KhError, match=text) as e:
        call(args)
    assert e.value.status == 1


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 2}, "dtype"), ({"head_dim": 63}, "head_dim"), ({"head_dim": 0}, "head_dim"), ({"head_dim": 258}, "head_dim"),
    ({"rotary_dim": 66}, "rotary_dim"), ({"rotary_dim": 31}, "rotary_dim"), ({"rotary_dim": -2}, "rotary_dim"),
    ({"q_heads": 0, "k_heads": 0}, "heads"), ({"q_heads": -1}, "heads"), ({"q_heads": 4096, "k_heads": 1}, "heads"),
    ({"interleaved": 2}, "interleaved"), ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"rows": -1}, "rows"),
    ({"x_stride": 255}, "stride"), ({"out_stride": 255}, "stride"), ({"x": None}, "null"), ({"out": None}, "null"),
    ({"cossin": None}, "null"), ({"positions": None}, "null"), ({"table_rows": 0}, "table_rows"),
    ({"x": P + 1}, "aligned"), ({"positions": P + 2}, "aligned"), ({"k_weight": P + 2}, "aligned"),
    ({"out": P + 512}, "overlaps"), ({"out": P, "out_stride": 512}, "overlaps"),
    ({"x_stride": 512, "out_stride": 512, "out": P + 500}, "overlaps"),
])
def test_norm_refusals(kw, text):
    refused(kb.qk_norm_rope, norm(**kw), text)


@pytest.mark.parametrize("kw,text", [
    ({"n_seqs": -1}, "n_seqs"), ({"n_seqs": 65536}, "n_seqs"), ({"head_dim": 48}, "head_dim"), ({"head_dim": 0}, "head_dim"),
    ({"q_heads": 3}, "q_heads"), ({"kv_heads": 0}, "kv_heads"), ({"q_heads": 0}, "q_heads"),
    ({"q_heads": 130, "kv_heads": 2}, "q_heads"), ({"max_q": -1}, "max_q"), ({"max_k": 1 << 25}, "max_k"),
    ({"q_rows": -1}, "rows"), ({"kv_rows": 1 << 31}, "rows"), ({"q": None}, "null"), ({"k": None}, "null"),
    ({"out": None}, "null"), ({"q_starts": None}, "null"), ({"k_starts": None}, "null"), ({"q": P + 8}, "aligned"),
    ({"v": P + 2}, "aligned"), ({"q_stride": 248}, "stride"), ({"k_stride": 120}, "stride"), ({"v_stride": 132}, "stride"),
    ({"out_stride": 252}, "stride"), ({"workspace": P + 64}, "workspace"),
    ({"scale": 0.0}, "scale"), ({"scale": -0.125}, "scale"), ({"scale": float("inf")}, "scale"),
    ({"scale": float("nan")}, "scale"), ({"q_heads": 1, "kv_heads": 1, "max_k": 9001, "workspace_bytes": 100}, "workspace"),
])
def test_cross_refusals(kw, text):
    refused(kb.cross_attention_f16, cross(**kw), text)


@pytest.mark.parametrize("kw,text", [
    ({"k": 60}, "k and n"), ({"n": 0}, "k and n"), ({"k": 65544}, "k and n"), ({"rank": 4}, "rank"), ({"rank": 136}, "rank"),
    ({"n_adapters": -1}, "n_adapters"), ({"n_segs": 65536}, "n_segs"), ({"rows": -1}, "rows"), ({"x": None}, "null"),
    ({"w": None}, "null"), ({"lora_b": None}, "null"), ({"seg_starts": None}, "null"), ({"seg_adapters": None}, "null"),
    ({"out": None}, "null"), ({"x": P + 2}, "aligned"), ({"bias": P + 8}, "aligned"), ({"x_stride": 56}, "stride"),
    ({"out_stride": 132}, "stride"), ({"workspace_bytes": 0}, "workspace"), ({"workspace": None}, "workspace"),
    ({"workspace": P + 128}, "workspace"),
])
def test_lora_refusals(kw, text):
    refused(kb.lora_matmul_f16, lora(**kw), text)


@pytest.mark.parametrize("call,args,text", [
    (kb.qk_norm_rope, norm(rows=1 << 31), "rows"),
    (kb.qk_norm_rope, norm(rows=(1 << 31) - 1, x_stride=(1 << 31) - 1), "stride"),
    (kb.qk_norm_rope, norm(x_stride=1 << 31), "stride"),
    (kb.lora_matmul_f16, lora(n=65528, n_adapters=32773), "n_adapters"),
    (kb.lora_matmul_f16, lora(n_adapters=65536), "n_adapters"),
    (kb.lora_matmul_f16, lora(rows=(1 << 31) - 256), "rows"),
    (kb.lora_matmul_f16, lora(x_stride=1 << 31), "stride"),
    (kb.lora_matmul_f16, lora(out=P), "out may not be x"),
    (kb.cross_attention_f16, cross(v_stride=1 << 31), "stride"),
])
def test_limits_and_aliases_are_refused(call, args, text):
    refused(call, args, text)


def test_lora_workspace_grows_with_the_rows_alone():
    for rows in (0, 1, 128, 129, 70000):
        for na, segs in ((1, 1), (40, 60000)):
            assert kb.lora_matmul_f16_workspace(lora(rows=rows, rank=16, n_adapters=na, n_segs=segs)) == rows * 32
    assert kb.lora_matmul_f16_workspace(lora(n_adapters=0)) == 0


def test_null_arguments_are_refused():
    lib = kb.load_library()
    for name in ("kh_qk_norm_rope", "kh_cross_attention_f16", "kh_lora_matmul_f16"):
        assert getattr(lib, name)(None, None) == 1
        assert name in lib.kh_last_error().decode()
    for name in ("kh_cross_attention_f16_workspace", "kh_lora_matmul_f16_workspace"):
        assert getattr(lib, name)(None) == -1


def test_nothing_to_do_needs_no_device():
    kb.qk_norm_rope(norm(rows=0, x=None, out=None))
    kb.cross_attention_f16(cross(n_seqs=0, q=None, out=None))
    kb.cross_attention_f16(cross(max_q=0))
    kb.cross_attention_f16(cross(q_rows=0, q=None, out=None))
    kb.lora_matmul_f16(lora(n_segs=0))
    kb.lora_matmul_f16(lora(rows=0, x=None, out=None))


def test_struct_layout_matches_the_header(tmp_path):
    """The ctypes structures have the C compiler's sizes and offsets."""
    import re
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "kh_cuda.h"
    pairs = [("kh_qk_norm_rope_args", kb.QkNormRopeArgs), ("kh_cross_attention_args", kb.CrossAttentionArgs),
             ("kh_lora_matmul_args", kb.LoraMatmulArgs)]
    src = f'#include "{header}"\n#include <stdio.h>\nint main(void) {{\n'
    for name, st in pairs:
        src += f'printf("%zu\\n", sizeof({name}));\n'
        for f, _ in st._fields_:
            src += f'printf("%zu\\n", offsetof({name}, {f}));\n'
    src += "return 0; }\n"
    c = tmp_path / "layout.c"
    c.write_text(src)
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(c), "-o", str(tmp_path / "layout")], check=True)
    got = list(map(int, re.findall(r"\d+", subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True).stdout)))
    want = []
    for _, st in pairs:
        want.append(ctypes.sizeof(st))
        want += [getattr(st, f).offset for f, _ in st._fields_]
    assert got == want
