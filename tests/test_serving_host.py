"""The ragged step's argument checks, which need no GPU, and the restatements that its
GPU tests compare with, against one another on small cases."""
import os
import shutil
import struct
import subprocess

import pytest
import torch

from gqa_kernels import (RaggedPagedAttention, paged_ragged_attention, plan_step, qk_norm_rope, qk_norm_rope_append, rope_table,
                         verify_drafts, verify_drafts_greedy)
from tests._serving import plan64, rope64, verify64

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def attn(**kw):
    a = dict(query=bf(3, 8, 128), key_cache=bf(4, 64, 2, 128), value_cache=bf(4, 64, 2, 128), block_tables=i32(2, 2),
             cu_query_lens=i32(3), seq_lens=i32(2))
    a.update(kw)
    return paged_ragged_attention(**a)


@pytest.mark.parametrize("kw", [
    dict(query=bf(3, 8)), dict(query=bf(3, 7, 128)), dict(query=bf(3, 8, 64)), dict(value_cache=bf(4, 32, 2, 128)),
    dict(block_tables=i32(3, 2)), dict(cu_query_lens=i32(2)), dict(window=0), dict(softcap=-1.0),
    dict(causal=False, window=4), dict(causal=False, prefix_lens=i32(2))])
def test_attention_refuses(lib_path, kw):
    with pytest.raises(ValueError):
        attn(**kw)


@pytest.mark.parametrize("kw,err", [
    (dict(query=torch.zeros(3, 8, 128)), RuntimeError), (dict(key_cache=torch.zeros(4, 64, 2, 128)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError), (dict(), ValueError)])
def test_attention_types_and_devices(lib_path, kw, err):
    with pytest.raises(err):  # the last: tensors on the CPU
        attn(**kw)


def rope(**kw):
    a = dict(q=bf(3, 8, 128), k=bf(3, 2, 128), v=bf(3, 2, 128), positions=i32(3), cos_sin=torch.zeros(10, 128),
             key_cache=bf(4, 16, 2, 128), value_cache=bf(4, 16, 2, 128), slot_mapping=torch.zeros(3, dtype=torch.int64))
    a.update(kw)
    return qk_norm_rope_append(**a)


@pytest.mark.parametrize("kw", [
    dict(q=bf(3, 8, 96)), dict(k=bf(2, 2, 128), v=bf(2, 2, 128)), dict(positions=i32(4)), dict(positions=i32(5, 3)),
    dict(positions=i32(2, 3)), dict(positions=i32(2, 3), sections=[30, 30]), dict(cos_sin=torch.zeros(10, 24)),
    dict(cos_sin=torch.zeros(10, 256)), dict(q_weight=bf(64)), dict(key_cache=bf(4, 16, 3, 128), value_cache=bf(4, 16, 3, 128)),
    dict(out=bf(3, 8, 64)), dict()])
def test_rope_refuses(lib_path, kw):
    with pytest.raises(ValueError):
        rope(**kw)


@pytest.mark.parametrize("kw", [dict(slot_mapping=i32(3)), dict(value_cache=torch.zeros(4, 16, 2, 128)), dict(k=torch.zeros(3, 2, 128),
                                                                                                    v=torch.zeros(3, 2, 128))])
def test_rope_types(lib_path, kw):
    with pytest.raises(TypeError):
        rope(**kw)


def test_rope_without_cache_refuses(lib_path):
    with pytest.raises(ValueError):
        qk_norm_rope(bf(3, 8, 128), bf(3, 2, 64), i32(3), torch.zeros(9, 128))


@pytest.mark.parametrize("at,value,err", [
    (0, i32(3), ValueError), (2, i32(2), ValueError), (5, i32(2), ValueError), (3, torch.zeros(2, dtype=torch.int64), TypeError),
    (6, 24, ValueError), (7, -1, ValueError), (0, i32(2), ValueError)])
def test_plan_refuses(lib_path, at, value, err):
    args = [i32(2), i32(2), i32(2, 4), i32(2), i32(5), i32(1), 16, 8]
    args[at] = value
    with pytest.raises(err):
        plan_step(*args)


def verify(**kw):
    a = dict(draft_tokens=i32(2, 3), target_probs=torch.zeros(8, 50), draft_probs=torch.zeros(2, 3, 50),
             uniforms=torch.zeros(2, 3), exponentials=torch.zeros(2, 50), cu_query_lens=i32(3))
    a.update(kw)
    return verify_drafts(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(draft_tokens=i32(2, 65)), ValueError), (dict(cu_query_lens=i32(2)), ValueError), (dict(uniforms=torch.zeros(2, 2)), ValueError),
    (dict(exponentials=torch.zeros(2, 49)), ValueError), (dict(draft_probs=torch.zeros(2, 3, 49)), ValueError),
    (dict(draft_probs=bf(2, 3, 50)), TypeError), (dict(target_probs=torch.zeros(8, 50, dtype=torch.float64)), TypeError),
    (dict(draft_tokens=torch.zeros(2, 3, dtype=torch.int64)), TypeError), (dict(exponentials=None), ValueError),
    (dict(draft_tokens=[1]), TypeError), (dict(), ValueError)])
def test_verify_refuses(lib_path, kw, err):
    with pytest.raises(err):
        verify(**kw)


def test_greedy_refuses(lib_path):
    with pytest.raises(ValueError):
        verify_drafts_greedy(i32(2, 1), torch.zeros(4, 9), i32(3))  # on the CPU


def test_layer_refuses():
    with pytest.raises(ValueError):
        RaggedPagedAttention(7, 2, 128, rope_table(4, 128, device="cpu"))
    with pytest.raises(ValueError):
        RaggedPagedAttention(8, 2, 128, rope_table(4, 128, device="cpu"), kv_cache_dtype="int8")


# The structs' fields in order, as an FFI host packs them.
STEP_PLAN = struct.Struct("@14Pq5i").pack
QK_NORM_ROPE = struct.Struct("@11P10q16i3f").pack
RAGGED = struct.Struct("@PN11P14q14i4f").pack
VERIFY = struct.Struct("@PN8P6q5i").pack


def test_c_entry_points_refuse_before_any_launch(lib_path):
    """The C ABI's own checks answer with a status, on a machine without a GPU."""
    from gqa_kernels import _lib
    lib = _lib.load()
    one = 1 << 20  # a non-null, aligned address that is never read

    def ragged(hq=8, hkv=2, d=128, block=64, dtype=1, fp8=0, causal=1, window=0, scale=0.1, cap=0.0, table=one, max_len=64,
               dstr=1, n=1):
        return lib.gqa_ragged_fwd(RAGGED(0, 0,
            one, one, one, one, 0, table, one, one, 0, 0, 0, 8, 8, 1, 8, 8, 8, dstr, 8, 8, 8, 1, 8, 8, 1,
            1, n, 1, hq, hkv, d, block, 4, 1, max_len, window, causal, dtype, fp8, scale, cap, 1.0, 1.0), None)
    assert ragged(hq=7) == 1 and ragged(d=96) == 2 and ragged(hq=130) == 2 and ragged(block=8) == 2 and ragged(block=48) == 2
    assert ragged(dtype=5) == 2 and ragged(d=64, fp8=1) == 2 and ragged(causal=0, window=3) == 1 and ragged(window=-1) == 1
    assert ragged(scale=float("nan")) == 1 and ragged(cap=-1.0) == 1 and ragged(table=0) == 1 and ragged(max_len=65) == 1
    assert ragged(dstr=2) == 3 and ragged(n=0) == 0 and lib.gqa_ragged_fwd(None, None) == 1

    def plan(held_out=2 * one, block=16, stride=4):
        return lib.gqa_step_plan(STEP_PLAN(one, one, one, one, one, one, one, 3 * one, one, one, one, one, held_out, 2 * one,
                                                    stride, 2, 4, 4, block, 8), None)
    assert plan(held_out=one) == 1 and plan(block=12) == 2 and plan(stride=3) == 1 and lib.gqa_step_plan(None, None) == 1

    def rotate(d=128, rot=128, axes=1, sections=(64, 0, 0, 0), slots=one, eps=1e-6, q=one):
        return lib.gqa_qk_norm_rope(QK_NORM_ROPE(q, one, one, 0, 0, one, one, one, one, one, slots, 8, 8, 1, 8, 8, 1, 8, 8, 1, 0,
                                                          *sections, axes, 9, rot, 0, 3, 8, 2, d, 16, 4, 1, 0, eps, 1.0, 1.0), None)
    assert rotate(d=80) == 2 and rotate(rot=24) == 2 and rotate(axes=5) == 2 and rotate(axes=2, sections=(60, 3, 0, 0)) == 1
    assert rotate(slots=0) == 1 and rotate(eps=-1.0) == 1 and rotate(q=one + 8) == 3 and lib.gqa_qk_norm_rope(None, None) == 1

    def check(k=2, vocab=9, dtype=2, n=1):
        return lib.gqa_verify_drafts(VERIFY(0, 0, one, one, 0, one, one, one, one, one, 2, 9, 0, 0, 2, 9,
                                                                                 n, 3, k, vocab, dtype), None)
    assert check(k=65) == 2 and check(vocab=0) == 1 and check(dtype=7) == 2 and check(n=20000) == 2 and check(n=0) == 0
    assert lib.gqa_verify_drafts(None, None) == 1 and lib.gqa_verify_greedy(None, None) == 1


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_packed_structs_match_the_header(tmp_path):
    """The structs as a C compiler lays them out have the packed records' sizes and last fields' places."""
    want = {"gqa_step_plan_args": ("max_tokens", STEP_PLAN(*[0] * 20)), "gqa_qk_norm_rope_args": ("v_scale", QK_NORM_ROPE(*[0] * 40)),
            "gqa_ragged_args": ("v_scale", RAGGED(*[0] * 45)), "gqa_verify_args": ("dtype", VERIFY(*[0] * 21))}
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "gqa_sm100.h"\nint main(void) {\n' + "".join(
        f'  printf("%zu %zu\\n", sizeof({t}), offsetof({t}, {f}));\n' for t, (f, _) in want.items()) + "  return 0;\n}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [tuple(map(int, x.split())) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()]
    for (name, (_, packed)), (size, last) in zip(want.items(), got):
        assert last == len(packed) - 4 and -(-len(packed) // 8) * 8 == size, name


# ----------------------------------------------------------------------------- the restatements themselves
def test_rotation_keeps_lengths_and_turns_by_the_difference():
    """Rotated pairs keep their norm, and q.k depends on the positions' difference only."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 1, 64, generator=g).double()
    table = rope_table(200, 64, device="cpu").double()
    for inter in (False, True):
        def at(p, y=x):
            return rope64(y, None, 0.0, table[p:p + 1, :32], table[p:p + 1, 32:], inter)[0, 0]
        assert abs(float(at(150).norm() - x.norm())) < 1e-6
        assert abs(float(at(10) @ at(17) - at(110) @ at(117))) < 1e-5


def test_plan_restatement():
    out, table, left = plan64([3, 2, 0, 9], [6, 0, 4, 0], [[5, 6, -1], [-1] * 3, [7, -1, -1], [-1] * 3], [2, 0, 1, 0], [1, 2, 3], 2, 4, 16)
    assert out["granted"] == [True, True, True, False] and table[0] == [5, 6, 2] and table[1][0] == 1 and left == 0
    assert out["slot"][:5] == [6 * 4 + 2, 6 * 4 + 3, 2 * 4, 4, 5] and out["slot"][5:14] == [-1] * 9 and out["seq"] == [9, 2, 4, 0]


def test_verification_restatement_of_a_perfect_draft():
    p = torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7]])
    tok, num = verify64([[0]], p, p[None, :1], torch.tensor([[0.999]]), torch.ones(1, 3), [0, 2])
    assert tok == [[0, 2]] and num == [2]
