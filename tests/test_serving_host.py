"""Host side of the operators before and behind the attention, without a GPU: refusals and launch rules."""
from __future__ import annotations

import ctypes

import pytest
import torch

from conftest import import_submodule
from host_query import query

_lib = import_submodule("_lib")

BASE = 1 << 24
P = [ctypes.c_void_p(BASE * (i + 1)) for i in range(10)]  # never dereferenced: every call below fails validation
U, V = ctypes.c_void_p(BASE + 4), ctypes.c_void_p(BASE + 2)


def _calls(name, good, bad):
    for change, code in bad:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        yield pytest.param(name, args, code, id=f"{name}-{change}")


BAD = [
    # q, k, wq, wk, table, positions, qo, ko, T, n_q, n_kv, d, rot, rows, strides q k qo ko, eps, neighbours, dtype, stream
    *_calls("mx_qk_norm_rope", [*P[:8], 5, 4, 2, 64, 32, 100, 512, 512, 256, 128, 1e-6, 0, 0, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in range(8)], *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(8, 14)],
        ({11: 40}, _lib.MX_ERR_SHAPE), ({11: 272, 12: 16}, _lib.MX_ERR_SHAPE), ({12: 80}, _lib.MX_ERR_SHAPE),
        ({12: 24}, _lib.MX_ERR_SHAPE), ({14: 248}, _lib.MX_ERR_SHAPE), ({15: 120}, _lib.MX_ERR_SHAPE),
        ({16: 248}, _lib.MX_ERR_SHAPE), ({17: 120}, _lib.MX_ERR_SHAPE), ({9: 2 ** 26}, _lib.MX_ERR_SHAPE), ({8: 2 ** 29}, _lib.MX_ERR_SHAPE),
        *[({i: 516}, _lib.MX_ERR_ALIGN) for i in (14, 15, 16, 17)],
        *[({i: U}, _lib.MX_ERR_ALIGN) for i in (0, 1, 2, 3, 4, 6, 7)], ({5: V}, _lib.MX_ERR_ALIGN),
        ({20: 2}, _lib.MX_ERR_DTYPE), ({6: P[1]}, _lib.MX_ERR_ALIAS), ({7: P[0]}, _lib.MX_ERR_ALIAS),
        ({6: P[0]}, _lib.MX_ERR_ALIAS),  # q's memory at another stride
        ({7: P[6]}, _lib.MX_ERR_ALIAS)]),
    # q, kc, vc, ks, vs, table, lens, cu, O, B, T, max_q, max_kv, n_q, n_kv, d, page, pages, max_pages, ldq, scale, window,
    # sinks, dtype, workspace, bytes, stream
    *_calls("mx_gqa_kv8_window", [P[0]] * 9 + [2, 5, 4, 4096, 4, 2, 64, 16, 9, 300, 256, 0.1, 3000, 4, 0, P[0], 1 << 30, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in (0, 1, 2, 3, 4, 5, 6, 8)], ({7: None}, _lib.MX_ERR_SHAPE),
        *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(9, 19)], ({13: 5}, _lib.MX_ERR_SHAPE), ({15: 96}, _lib.MX_ERR_SHAPE),
        ({19: 248}, _lib.MX_ERR_SHAPE), ({19: 260}, _lib.MX_ERR_ALIGN), ({0: U}, _lib.MX_ERR_ALIGN),
        ({21: 0}, _lib.MX_ERR_SHAPE), ({21: -1}, _lib.MX_ERR_SHAPE), ({22: -1}, _lib.MX_ERR_SHAPE),
        ({23: 2}, _lib.MX_ERR_DTYPE), ({24: None}, _lib.MX_ERR_WORKSPACE), ({25: 1000}, _lib.MX_ERR_WORKSPACE),
        ({24: U}, _lib.MX_ERR_ALIGN)]),
    # q, kc, vc, ks, vs, table, lens, cu, tree, O, B, T, max_q, max_kv, n_q, n_kv, d, page, pages, max_pages, ldq, scale,
    # words, dtype, workspace, bytes, stream
    *_calls("mx_gqa_kv8_tree", [P[0]] * 10 + [2, 5, 4, 4096, 4, 2, 64, 16, 9, 300, 256, 0.1, 1, 0, P[0], 1 << 30, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in (0, 1, 2, 3, 4, 5, 6, 8, 9)], ({7: None}, _lib.MX_ERR_SHAPE),
        *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(10, 20)], ({14: 5}, _lib.MX_ERR_SHAPE), ({16: 96}, _lib.MX_ERR_SHAPE),
        ({20: 248}, _lib.MX_ERR_SHAPE), ({20: 260}, _lib.MX_ERR_ALIGN), ({8: U}, _lib.MX_ERR_ALIGN),
        ({22: 0}, _lib.MX_ERR_SHAPE), ({22: 17}, _lib.MX_ERR_SHAPE), ({23: 2}, _lib.MX_ERR_DTYPE),
        ({24: None}, _lib.MX_ERR_WORKSPACE), ({25: 1000}, _lib.MX_ERR_WORKSPACE), ({24: U}, _lib.MX_ERR_ALIGN)]),
    # logits, tokens, logprob, entropy, ids, top_logprob, T, V, stride, given, top, dtype, workspace, bytes, stream
    *_calls("mx_token_logprobs", [*P[:6], 3, 50000, 50000, 2, 5, 0, P[6], 1 << 24, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in range(6)], ({6: 0}, _lib.MX_ERR_SHAPE), ({7: 0}, _lib.MX_ERR_SHAPE),
        ({7: 2 ** 30 + 1, 8: 2 ** 30 + 1}, _lib.MX_ERR_SHAPE), ({8: 49999}, _lib.MX_ERR_SHAPE), ({8: 2 ** 31}, _lib.MX_ERR_SHAPE),
        ({9: -1}, _lib.MX_ERR_SHAPE), ({10: -1}, _lib.MX_ERR_SHAPE), ({10: 33}, _lib.MX_ERR_SHAPE),
        ({7: 4, 8: 4}, _lib.MX_ERR_SHAPE), ({6: 2 ** 30}, _lib.MX_ERR_SHAPE), ({11: 3}, _lib.MX_ERR_DTYPE),
        ({0: ctypes.c_void_p(BASE + 1)}, _lib.MX_ERR_ALIGN), ({0: V, 11: 2}, _lib.MX_ERR_ALIGN),
        *[({i: V}, _lib.MX_ERR_ALIGN) for i in range(1, 6)], ({12: None}, _lib.MX_ERR_WORKSPACE),
        ({13: 100}, _lib.MX_ERR_WORKSPACE), ({12: U}, _lib.MX_ERR_ALIGN)]),
]


@pytest.mark.parametrize("name,args,code", BAD)
def test_entry_points_refuse(name, args, code):
    assert getattr(_lib.load(), name)(*args) == code


def test_logprob_slices(tmp_path):
    """Every block of a row, at whichever alignment, lies in one slice; no slice is empty; a wave's lanes hold them all."""
    out = query(tmp_path, "token_logprobs.hip", r"""
  using namespace mx::logprobs;
  for (int T : {1, 2, 17, 64, 511, 512, 100000, 1 << 30})
    for (int V : {1, 3, 8, 4095, 4096, 32000, 100003, 200000, 1 << 30})
      for (int dtype : {MX_DTYPE_BF16, MX_DTYPE_F32}) {
        const Plan p = plan(T, V, dtype);
        const long long blocks = V / (dtype == MX_DTYPE_F32 ? 4 : 8);
        const bool whole = (long long)p.slices * p.per >= blocks, used = p.slices == 1 || (p.slices - 1LL) * p.per < blocks;
        if (!whole || !used || p.slices < 1 || p.slices > kMostSlices || p.per < 1) printf("plan(%d, %d, %d)\n", T, V, dtype);
      }
  printf("%d %d\n", plan(1, 32000, MX_DTYPE_BF16).threads, plan(1, 50000, MX_DTYPE_BF16).slices > 1);""")
    assert out == ["1024 1"]


def test_attention_plans(tmp_path):
    """Windows and trees over many sizes: the splits cover what a block of rows may visit and none starts behind it, a chunk is
    whole tiles where there are several, and a tree's workgroups hold its rows."""
    window = query(tmp_path, "kv8_window.hip", r"""
  using namespace mx::kv8;
  for (int B : {1, 3, 64, 4096})
    for (int T : {1, 17, 33, 1000, 100000})
      for (int kv : {1, 255, 1000, 8192, 1 << 30})
        for (int G : {1, 4, 48})
          for (int w : {1, 64, 1000, 4096, 2147483647})
            for (int s : {0, 4, 200, 2147483647}) {
              const int d = T % 2 ? 64 : 128;
              const Plan p = window_plan(B, T, T, kv, 2 * G, 2, d, w, s);
              const long long view = std::min<long long>(kv, 64 * (up(s, 64) + up((long long)w + std::min(T, 32) + 62, 64)));
              const bool whole = p.splits >= 1 && p.splits <= 65535 && p.chunk >= 1 && (p.splits == 1 || p.chunk % 64 == 0);
              if (!whole || (p.splits > 1 && (long long)(p.splits - 1) * p.chunk >= view))
                printf("window_plan(%d, %d, %d, %d, %d, %d)\n", B, T, kv, G, w, s);
            }
  printf("ok\n");""")
    tree = query(tmp_path, "kv8_tree.hip", r"""
  using namespace mx::kv8;
  for (int B : {1, 3, 64, 4096})
    for (int T : {1, 17, 33, 64, 100, 257, 100000})
      for (int kv : {1, 255, 1000, 8192, 1 << 30})
        for (int G : {1, 4, 48})
          for (int d : {64, 128}) {
            const Plan p = tree_plan(B, T, T, kv, 2 * G, 2, d);
            const long long rows = (long long)T * G;
            const bool fits = p.nr ? rows <= 16LL * p.nr * p.blocks && p.blocks <= 65535 : p.tiles == std::min(up(rows, 32 * p.waves), 65535LL);
            const bool whole = p.splits >= 1 && p.splits <= 65535 && p.chunk >= 1 && (p.splits == 1 || p.chunk % 64 == 0);
            if (!fits || !whole || (p.splits > 1 && (long long)(p.splits - 1) * p.chunk >= kv) || (p.waves == 4 && d != 64))
              printf("tree_plan(%d, %d, %d, %d, %d)\n", B, T, kv, G, d);
          }
  for (int d : {64, 128}) {  // tiles, which split long contexts, blocks of 16 and of 32, one block of 32
    const Plan a = tree_plan(603, 98, 64, 300, 4, 1, d), b = tree_plan(140, 98, 64, 5000, 4, 1, d);
    const Plan c = tree_plan(1, 13, 13, 1001, 32, 8, d), e = tree_plan(123, 39, 13, 1000, 4, 1, d), f = tree_plan(123, 24, 8, 4000, 4, 1, d);
    if (a.nr || a.splits != 1 || b.nr || b.splits < 2 || c.nr != 1 || c.blocks != 4 || e.nr != 2 || e.blocks != 2 || f.nr != 2 ||
        f.blocks != 1)
      printf("d %d\n", d);
  }
  printf("ok\n");""")
    assert window == ["ok"] and tree == ["ok"]


def test_workspaces():
    lib = _lib.load()
    assert lib.mx_gqa_kv8_window_workspace(1, 1, 1, 100000, 32, 8, 128, 512, 4) > 0
    assert lib.mx_gqa_kv8_window_workspace(1, 1, 1, 100000, 32, 8, 64, 1000, 4) == 0  # one workgroup
    assert lib.mx_gqa_kv8_window_workspace(1, 1, 1, 100000, 32, 8, 128, 0, 4) == 0
    assert lib.mx_gqa_kv8_tree_workspace(1, 13, 13, 1001, 32, 8, 128) > 0
    assert lib.mx_gqa_kv8_tree_workspace(1, 13, 13, 1001, 31, 8, 128) == 0
    f = lib.mx_token_logprobs_workspace
    assert f(1000, 50000, 5, 0) == 0 and f(1, 100, 5, 0) == 0 and f(2, 50000, 5, 0) > 0
    assert [f(*a) for a in ((0, 50000, 5, 0), (1, 0, 0, 0), (1, 50000, 33, 0), (1, 50000, 5, 4))] == [0] * 4


def test_operators_refuse_before_the_device():
    """Types and devices that the operators check by themselves: CPU tensors reach no kernel."""
    ops = import_submodule("ops")
    q, k, w = torch.zeros(2, 4, 64), torch.zeros(2, 1, 64), torch.ones(64)
    table, places = ops.rope_table(8, 32, device="cpu"), torch.zeros(2, dtype=torch.int32)
    bf = torch.bfloat16
    for call in (lambda: ops.qk_norm_rope(q.to(bf), k.to(bf), w.to(bf), w.to(bf), table, places),
                 lambda: ops.token_logprobs(w[None]), lambda: ops.token_logprobs(w[None].to(bf), places[:1], top=3)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    for call in (lambda: ops.qk_norm_rope(q, k, w, w, table, places), lambda: ops.token_logprobs(places[None]),
                 lambda: ops.token_logprobs([1.0]), lambda: ops.gqa_kv8_window(q.to(bf), None, places, places, 4),
                 lambda: ops.gqa_kv8_tree(q.to(bf), None, places, places, places)):
        with pytest.raises(TypeError):
            call()
    for window, sinks in ((0, 0), (-1, 0), (1 << 31, 0), (4, -1), (4, 1 << 31)):
        with pytest.raises(ValueError, match="window"):
            ops.gqa_kv8_window(q.to(bf), None, places, places, window, sinks)
    for positions, rot in ((0, 32), (8, 24), (8, 0)):
        with pytest.raises(ValueError, match="multiple of 16"):
            ops.rope_table(positions, rot, device="cpu")


@pytest.mark.parametrize("words", [(1 << 30) + 1, (1 << 30) + 8, (1 << 31) - 1])
def test_tree_words_past_half_of_an_int(words):
    """Counts whose double, in words of 32 bits, leaves an int's range: refused like any other past 16."""
    args = [P[0]] * 10 + [2, 5, 4, 4096, 4, 2, 64, 16, 9, 300, 256, 0.1, words, 0, P[0], 1 << 30, None]
    assert _lib.load().mx_gqa_kv8_tree(*args) == _lib.MX_ERR_SHAPE


def test_windows_of_one_workgroup(tmp_path):
    """The rule for one workgroup on both head sizes, past what the causal form keeps to one; what a tile block visits past the
    count that sizes the splits."""
    out = query(tmp_path, "kv8_window.hip", r"""
  using namespace mx::kv8;
  for (int d : {64, 128})
    for (int w = 1; w < 3000; ++w)
      for (int s : {0, 4, 100}) {
        const Plan p = window_plan(1, 1, 1, 100000, 8, 2, d, w, s);
        const long long kv = 64 * (up(s, 64) + up(w + 63, 64));
        if ((p.splits == 1) != (kv * d <= 65536 + 8192)) printf("d %d window %d sinks %d\n", d, w, s);
        const long long tiles = up(w + 256 + 62, 64) - up(w + 32 + 62, 64);
        if (tiles < 3 || tiles > 4) printf("window %d: %lld tiles\n", w, tiles);
      }
  printf("%d %d\n", window_plan(1, 1, 1, 100000, 8, 2, 64, 1024, 64).splits, window_plan(1, 1, 1, 100000, 8, 2, 128, 449, 64).splits);""")
    assert out == ["1 1"]


def test_plans_of_the_wide_forms(tmp_path):
    """128 channels: split keys in blocks of 32 rows side by side, and tiles with and without a split (as tests on the GPU
    take them)."""
    window = query(tmp_path, "kv8_window.hip", r"""
  using namespace mx::kv8;
  const Plan a = window_plan(3, 35, 13, 8300, 32, 8, 128, 7000, 100), b = window_plan(140, 98, 64, 5000, 4, 1, 128, 2500, 100);
  const Plan c = window_plan(602, 140, 70, 300, 4, 1, 128, 150, 20), e = window_plan(602, 400, 200, 300, 1, 1, 128, 150, 20);
  printf("%d %d %d  %d %d  %d %d  %d %d\n", a.nr, a.blocks, a.splits > 1, b.nr, b.splits > 1, c.nr, c.splits, e.nr, e.splits);""")
    tree = query(tmp_path, "kv8_tree.hip", r"""
  using namespace mx::kv8;
  const Plan a = tree_plan(3, 35, 13, 8300, 32, 8, 128), b = tree_plan(140, 98, 64, 5000, 4, 1, 128);
  const Plan c = tree_plan(603, 180, 60, 300, 4, 1, 128), e = tree_plan(1, 13, 13, 32768, 32, 8, 128);
  printf("%d %d %d  %d %d  %d %d  %d %d %d\n", a.nr, a.blocks, a.splits > 1, b.nr, b.splits > 1, c.nr, c.splits, e.nr, e.blocks, e.splits);""")
    assert window == ["2 2 1  0 1  0 1  0 1"] and tree == ["2 2 1  0 1  0 1  2 2 16"]
