"""Paged key-value cache without a GPU: what the Python layer and the C entry points refuse, and that the
packed arguments have the layout of the C structs."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest
import torch

import paged_ref as R
from syncopate_b200 import _lib as L
from syncopate_b200.computation.paged import _interleaved, page_plan, paged_append, paged_attention
from syncopate_b200.operators import PagedKVCache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = dict(dtype=torch.int32)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_packed_arguments_have_the_layout_of_the_c_structs(tmp_path):
    structs = {"syn_page_plan_args": L.PagePlanArgs, "syn_paged_append_args": L.PagedAppendArgs,
               "syn_paged_attn_args": L.PagedAttnArgs}
    spelled = {"k_stride_token": "k_strides[0]", "k_stride_head": "k_strides[1]", "v_stride_token": "v_strides[0]",
               "v_stride_head": "v_strides[1]", "q_stride_token": "q_strides[0]", "q_stride_head": "q_strides[1]",
               "o_stride_token": "o_strides[0]", "o_stride_head": "o_strides[1]", "cache_stride_page": "cache_strides[0]",
               "cache_stride_slot": "cache_strides[1]", "cache_stride_head": "cache_strides[2]"}
    lines = ['#include "syncopate_b200.h"', "#include <stdio.h>", "int main(void) {"]
    want = []
    for name, cls in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {spelled.get(field, field)}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def _plan_tensors():
    return dict(lens=torch.zeros(3, **I32), add=torch.zeros(3, **I32), table=torch.zeros(3, 4, **I32),
                free_pages=torch.arange(8, **I32), num_free=torch.full((1,), 8, **I32), page_size=16, slots=torch.zeros(9, **I32),
                positions=torch.zeros(9, **I32), starts=torch.zeros(4, **I32))


@pytest.mark.parametrize("change, words", [
    (dict(lens=torch.zeros(2, **I32)), "one entry a row"),
    (dict(add=torch.zeros(3, dtype=torch.int64)), "add must be a contiguous int32"),
    (dict(table=torch.zeros(4, 3, **I32).t()), "unit inner stride"),
    (dict(table=torch.zeros(6, **I32).as_strided((3, 4), (1, 1))), "overlap"),
    (dict(starts=torch.zeros(3, **I32)), "starts one more"),
    (dict(positions=torch.zeros(8, **I32)), "same length"),
    (dict(num_free=torch.zeros(2, **I32)), "one number"),
    (dict(page_size=0), "page_size"),
    (dict(lens_out=torch.zeros(3)), "lens_out must be"),
    (dict(), "CUDA device"),
])
def test_page_plan_refuses(change, words):
    args = {**_plan_tensors(), **change}
    with pytest.raises(ValueError, match=words):
        page_plan(**args)


BF, HF, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def _append_tensors():
    return dict(k=torch.zeros(5, 2, 64, dtype=BF), v=torch.zeros(5, 2, 64, dtype=BF), slots=torch.zeros(5, **I32),
                k_cache=torch.zeros(4, 16, 2, 64, dtype=BF), v_cache=torch.zeros(4, 16, 2, 64, dtype=BF))


@pytest.mark.parametrize("change, words", [
    (dict(k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64)), "fp16/bf16"),
    (dict(v=torch.zeros(5, 2, 64, dtype=HF)), "fp16/bf16 tensors of one type"),
    (dict(v=torch.zeros(4, 2, 64, dtype=BF)), "one shape"),
    (dict(k=torch.zeros(5, 64, 2, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(slots=torch.zeros(4, **I32)), "4 slots for 5 tokens"),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), "slots must be"),
    (dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=BF).transpose(1, 2)), "same shape and strides"),
    (dict(k_cache=torch.zeros(4, 16, 2, 128, dtype=BF), v_cache=torch.zeros(4, 16, 2, 128, dtype=BF)), "heads and dim"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=HF), v_cache=torch.zeros(4, 16, 2, 64, dtype=HF)), "caches must be"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64).to(E4), v_cache=torch.zeros(4, 16, 2, 64).to(E4)), "needs k_scale"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64).to(E4), v_cache=torch.zeros(4, 16, 2, 64).to(E4), k_scale=torch.ones(2),
          v_scale=torch.ones(3)), "needs v_scale"),
    (dict(k_scale=torch.ones(2), v_scale=torch.ones(2)), "8-bit"),
    (dict(), "CUDA device"),
])
def test_paged_append_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        paged_append(**{**_append_tensors(), **change})


def _attend_tensors():
    return dict(q=torch.zeros(3, 4, 64, dtype=BF), k_cache=torch.zeros(4, 16, 2, 64, dtype=BF),
                v_cache=torch.zeros(4, 16, 2, 64, dtype=BF), table=torch.zeros(3, 2, **I32), lens=torch.zeros(3, **I32), sm_scale=1.0)


@pytest.mark.parametrize("change, words", [
    (dict(q=torch.zeros(3, 4, 64)), "fp16/bf16"),
    (dict(q=torch.zeros(3, 256, dtype=BF)), r"\[tokens, q_heads, dim\]"),
    (dict(q=torch.zeros(3, 4, 80, dtype=BF)), "head dimension"),
    (dict(q=torch.zeros(3, 64, 4, dtype=BF).transpose(1, 2)), "contiguous"),
    (dict(q=torch.zeros(3, 3, 64, dtype=BF)), "3 query heads over 2"),
    (dict(q=torch.zeros(3, 4, 128, dtype=BF)), "its head dimension"),
    (dict(q=torch.zeros(4, 4, 64, dtype=BF)), "pass starts"),
    (dict(lens=torch.zeros(2, **I32)), "lens needs"),
    (dict(table=torch.zeros(3, 2, dtype=torch.int64)), "table must be"),
    (dict(starts=torch.zeros(3, **I32)), "starts needs"),
    (dict(window=-1), "window"),
    (dict(window=4, causal=False), "window"),
    (dict(num_sms=-1), "num_sms"),
    (dict(out=torch.zeros(3, 4, 64, dtype=HF)), "out must have"),
    (dict(lse=torch.zeros(3, 4, dtype=BF)), "lse must be"),
    (dict(lse=torch.zeros(4, 3).t()), "lse must be"),
    (dict(k_scale=torch.ones(2)), "8-bit"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64).to(E4), v_cache=torch.zeros(4, 16, 2, 64).to(E4)), "needs k_scale"),
    (dict(), "CUDA device"),
])
def test_paged_attention_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        paged_attention(**{**_attend_tensors(), **change})


def test_paged_attention_refuses_an_output_over_its_input():
    args = _attend_tensors()
    with pytest.raises(ValueError, match="overlap"):
        paged_attention(**args, out=args["q"])


@pytest.mark.parametrize("change, words", [
    (dict(head_dim=80), "head_dim"),
    (dict(num_pages=0), "positive"),
    (dict(cache_dtype=torch.float32), "keeps"),
    (dict(cache_dtype=E4), "needs both"),
    (dict(k_scale=torch.ones(1, 2), v_scale=torch.ones(1, 2)), "8-bit"),
    (dict(cache_dtype=E4, k_scale=torch.ones(2), v_scale=torch.ones(2)), "layers, kv_heads"),
])
def test_cache_object_refuses(change, words):
    args = dict(num_pages=4, page_size=16, kv_heads=2, head_dim=64, max_requests=2, max_len=64, max_tokens=8, device="cpu")
    with pytest.raises(ValueError, match=words):
        PagedKVCache(**{**args, **change})


FAKE = 1 << 20  # never read: every call below is refused on the host


def _struct(cls, **changes):
    s = cls()
    for name, kind in cls._fields_:
        if kind is C.c_void_p:
            setattr(s, name, FAKE)
    for name, value in changes.items():
        setattr(s, name, value)
    return bytes(s)


def test_c_entry_points_refuse_on_the_host():
    lib = L.lib()
    assert lib.syn_page_plan(None, None) == lib.syn_paged_append(None, None) == lib.syn_paged_attention(None, None) == -1
    ok = dict(requests=2, width=4, page_size=16, num_pages=8, tokens=4, table_stride=4, device=-1)
    for change, code in [(dict(requests=0), -1), (dict(requests=8193), -9), (dict(table_stride=3), -1), (dict(slots=0), -1),
                         (dict(page_size=0), -1), (dict(tokens=-1), -1), (dict(lens=0), -1),
                         (dict(num_pages=1 << 20, page_size=1 << 12), -9)]:
        assert lib.syn_page_plan(_struct(L.PagePlanArgs, **{**ok, **change}), None) == code, change
    ok = dict(tokens=3, Hkv=2, D=64, page_size=16, num_pages=8, dtype=1, device=-1, k_stride_token=128, k_stride_head=64,
              v_stride_token=128, v_stride_head=64, cache_stride_page=2048, cache_stride_slot=128, cache_stride_head=64)
    for change, code in [(dict(D=72), -8), (dict(dtype=2), -8), (dict(cache_dtype=2), -8), (dict(k=FAKE + 2), -1),
                         (dict(k_stride_token=100), -1), (dict(cache_stride_slot=0), -1), (dict(cache_stride_page=-2048), -1),
                         (dict(cache_dtype=1, k_scale=0), -1), (dict(num_pages=1 << 28), -9), (dict(v=0), -1)]:
        assert lib.syn_paged_append(_struct(L.PagedAppendArgs, **{**ok, **change}), None) == code, change
    assert lib.syn_paged_append(_struct(L.PagedAppendArgs, **{**ok, "tokens": 0}), None) == 0
    ok = dict(k_scale=0, v_scale=0, tokens=3, requests=3, Hq=4, Hkv=2, D=64, page_size=16, num_pages=8, width=4, causal=1,
              table_stride=4, sm_scale=1.0, dtype=1, device=-1, q_stride_token=256, q_stride_head=64, o_stride_token=256,
              o_stride_head=64, cache_stride_page=2048, cache_stride_slot=128, cache_stride_head=64,
              workspace_bytes=1 << 40)
    for change, code in [(dict(D=96), -8), (dict(Hq=5), -1), (dict(starts=0, requests=2), -1), (dict(window=-1), -1),
                         (dict(window=3, causal=0), -1), (dict(dtype=3), -8), (dict(cache_dtype=3), -8), (dict(q=FAKE + 8), -1),
                         (dict(o_stride_head=60), -1), (dict(o_stride_token=0), -1), (dict(k_scale=FAKE), -1),
                         (dict(cache_dtype=1), -1), (dict(table_stride=3), -1), (dict(lens=0), -1), (dict(num_sms=-1), -1),
                         (dict(num_pages=1 << 28), -9)]:
        assert lib.syn_paged_attention(_struct(L.PagedAttnArgs, **{**ok, **change}), None) == code, change
    assert lib.syn_paged_attention(_struct(L.PagedAttnArgs, **{**ok, "tokens": 0}), None) == 0
    assert lib.syn_paged_attention_workspace(148, 128) > 0
    assert lib.syn_paged_attention_workspace(0, 128) == -1 and lib.syn_paged_attention_workspace(148, 96) == -8
    assert lib.syn_strerror(-10) != b"unknown error" and lib.syn_strerror(-11) != b"unknown error"


def test_the_reference_plan_by_hand():
    table = [[5, -1, -1], [7, 3, -1], [2, -1, -1]]
    slots, positions, starts, lens, top, table, free = R.plan([3, 8, 4], [2, -1, 1], table, [0, 1, 4, -1, -1, -1], 3, 4, 5)
    # Pages 7 and 3 go back, then request 0 takes 3 and request 2 takes 7.
    assert (slots, positions) == ([5 * 4 + 3, 3 * 4, 7 * 4, -1, -1], [3, 4, 4, 0, 0])
    assert (starts, lens, top, free) == ([0, 2, 2, 3], [5, 0, 5], 3, [0, 1, 4])
    assert [r[:2] for r in table] == [[5, 3], [7, 3], [2, 7]]


def _overlaps(name):
    """Arguments of paged_attention whose output shares memory with what is read."""
    args = _attend_tensors()
    T, H, D = 6, 4, 64
    args.update(table=torch.zeros(T, 2, **I32), lens=torch.zeros(T, **I32))
    flat = torch.zeros(64 * 1024, dtype=BF)
    wide = flat[: T * 3 * H * D].view(T, 3 * H, D)
    if name == "one head on":
        args.update(q=wide[:, 1: 1 + H], out=wide[:, 2: 2 + H])
    elif name == "one token on":
        args.update(q=flat[: T * H * D].view(T, H, D), out=flat[H * D: (T + 1) * H * D].view(T, H, D))
    elif name == "half a head on":
        args.update(q=flat[: T * H * D].view(T, H, D), out=flat[32: 32 + T * H * D].view(T, H, D))
    elif name == "other strides":
        args.update(q=wide[:, :H], out=flat[H * D: (T + 1) * H * D].view(T, H, D))
    elif name == "around the end of a row":  # its last heads lie on the next token's first ones
        args.update(q=wide[:, :H], out=flat[10 * D: 10 * D + T * 3 * H * D].view(T, 3 * H, D)[:, :H])
    elif name == "every other head":
        args.update(q=wide[:, 0: 2 * H: 2], out=wide[:, 2: 2 + 2 * H: 2])
    elif name in ("out on k_cache", "out on v_cache"):
        args.update(q=wide[:, :H], out=args[name[7:]].view(-1)[: T * H * D].view(T, H, D))
    elif name.startswith("lse"):
        args.update(q=flat[: T * H * D].view(T, H, D), out=flat[T * H * D: 2 * T * H * D].view(T, H, D))
        args["lse"] = args[name[7:]].reshape(-1)[-2 * T * H:].view(torch.float32).view(T, H)
    return args


@pytest.mark.parametrize("name", ["one head on", "one token on", "half a head on", "other strides", "around the end of a row",
                                  "every other head", "out on k_cache", "out on v_cache", "lse on q", "lse on out", "lse on k_cache",
                                  "lse on v_cache"])
def test_paged_attention_refuses_outputs_over_what_is_read(name):
    with pytest.raises(ValueError, match="must not overlap"):
        paged_attention(**_overlaps(name))


def test_paged_attention_takes_outputs_between_the_rows_of_its_input():
    # Refused for want of a GPU alone.
    T, H, D = 6, 4, 64
    flat = torch.zeros(64 * 1024, dtype=BF)
    wide = flat[: T * 3 * H * D].view(T, 3 * H, D)
    args = {**_attend_tensors(), "table": torch.zeros(T, 2, **I32), "lens": torch.zeros(T, **I32)}
    for q, out in [(wide[:, :H], wide[:, H: 2 * H]), (wide[:, H: 2 * H], wide[:, :H]), (wide[:, 2 * H:], wide[:, :H]),
                   (wide[:, 0: 2 * H: 2], wide[:, 1: 2 * H: 2]), (wide[::2, :H], wide[1::2, :H]),
                   (flat[: T * H * D].view(T, H, D), flat[T * H * D: 2 * T * H * D].view(T, H, D))]:
        n = q.shape[0]
        change = dict(q=q, out=out, table=args["table"][:n], lens=args["lens"][:n])
        with pytest.raises(ValueError, match="CUDA device"):
            paged_attention(**{**args, **change})


def test_outputs_taken_as_interleaved_share_no_element():
    rng, taken = random.Random(0), 0
    for _ in range(4000):
        shape = tuple(rng.randint(1, 4) for _ in range(3))
        strides = [(rng.choice([2, 4, 6, 8, 12, 16, 24, 32]), rng.choice([1, 2, 3, 4, 6, 8, 12]), 1) for _ in range(2)]
        if rng.random() < 0.7:
            strides[1] = strides[0]
        buf = torch.arange(400, dtype=torch.int32)
        a, b = (buf.as_strided(shape, s, rng.randint(0, 40)) for s in strides)
        if _interleaved(a, b):
            taken += 1
            assert not set(a.flatten().tolist()) & set(b.flatten().tolist()), (shape, strides)
    assert taken > 300
