"""The 8-bit operators' host side, without a GPU: refusals, the numbers that kernels take from the device
(compiled for the host from the kernels' own header), page bookkeeping."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from conftest import import_submodule
from host_query import query

_lib = import_submodule("_lib")
kv_pages = import_submodule("kv_pages")

P = ctypes.c_void_p(0x10000)  # never dereferenced: every call below fails validation
U = ctypes.c_void_p(0x10004)
V = ctypes.c_void_p(0x10002)


def _calls(name, good, bad):
    for change, code in bad:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        yield pytest.param(name, args, code, id=f"{name}-{change}")


BAD = [
    # X, Q, scales, M, K, ldx, dtype, stream
    *_calls("mx_quant_int8", [P, P, P, 4, 64, 64, 0, None], [
        ({0: None}, _lib.MX_ERR_NULL), ({1: None}, _lib.MX_ERR_NULL), ({2: None}, _lib.MX_ERR_NULL),
        ({3: 0}, _lib.MX_ERR_SHAPE), ({3: -1}, _lib.MX_ERR_SHAPE), ({4: 0, 5: 0}, _lib.MX_ERR_SHAPE),
        ({4: 40}, _lib.MX_ERR_SHAPE), ({5: 48}, _lib.MX_ERR_SHAPE), ({5: 68}, _lib.MX_ERR_ALIGN),
        ({0: U}, _lib.MX_ERR_ALIGN), ({1: U}, _lib.MX_ERR_ALIGN), ({2: V}, _lib.MX_ERR_ALIGN), ({6: 2}, _lib.MX_ERR_DTYPE)]),
    # A, sA, B, sB, C, M, N, K, dtype, stream
    *_calls("mx_gemm_int8", [P, P, P, P, P, 4, 8, 64, 0, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in range(5)], *[({i: 0}, _lib.MX_ERR_SHAPE) for i in (5, 6, 7)],
        ({7: 72}, _lib.MX_ERR_SHAPE), ({7: 131072}, _lib.MX_ERR_SHAPE), ({5: 2 ** 31 - 1, 6: 2 ** 31 - 1}, _lib.MX_ERR_SHAPE),
        *[({i: U}, _lib.MX_ERR_ALIGN) for i in (0, 2, 4)], *[({i: V}, _lib.MX_ERR_ALIGN) for i in (1, 3)],
        ({8: 3}, _lib.MX_ERR_DTYPE)]),
    # X, W, sW, C, M, N, K, ldx, dtype, workspace, bytes, stream
    *_calls("mx_linear_int8", [P, P, P, P, 40, 8, 64, 64, 0, P, 1 << 20, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in (0, 1, 2, 3, 9)], *[({i: 0}, _lib.MX_ERR_SHAPE) for i in (4, 5, 6)],
        ({4: -5}, _lib.MX_ERR_SHAPE), ({6: 72}, _lib.MX_ERR_SHAPE), ({7: 56}, _lib.MX_ERR_SHAPE),
        ({7: 68}, _lib.MX_ERR_ALIGN), ({0: U}, _lib.MX_ERR_ALIGN), ({9: U}, _lib.MX_ERR_ALIGN),
        ({8: 7}, _lib.MX_ERR_DTYPE), ({10: 2719}, _lib.MX_ERR_WORKSPACE), ({4: 8, 7: 2 ** 27}, _lib.MX_ERR_SHAPE),
        ({4: 1, 5: 2 ** 27}, _lib.MX_ERR_SHAPE)]),
    # k, v, kc, vc, ks, vs, table, lens, cu, B, T, max_q, n_kv, d, page, pages, max_pages, ldk, ldv, dtype, stream
    *_calls("mx_kv8_append", [P] * 9 + [2, 5, 4, 2, 64, 16, 9, 3, 128, 128, 0, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in range(8)], ({8: None}, _lib.MX_ERR_SHAPE),
        *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(9, 17)], ({13: 96}, _lib.MX_ERR_SHAPE), ({14: 48}, _lib.MX_ERR_SHAPE),
        ({14: 256}, _lib.MX_ERR_SHAPE), ({16: 2 ** 26 + 1}, _lib.MX_ERR_SHAPE), ({12: 2 ** 20, 9: 8}, _lib.MX_ERR_SHAPE),
        ({9: 2 ** 23 + 1}, _lib.MX_ERR_SHAPE), ({15: 2 ** 31 - 1}, _lib.MX_ERR_SHAPE),
        ({17: 120}, _lib.MX_ERR_SHAPE), ({18: 64}, _lib.MX_ERR_SHAPE), ({17: 132}, _lib.MX_ERR_ALIGN),
        ({18: 130}, _lib.MX_ERR_ALIGN), *[({i: U}, _lib.MX_ERR_ALIGN) for i in range(4)],
        *[({i: V}, _lib.MX_ERR_ALIGN) for i in (4, 5)], ({19: 2}, _lib.MX_ERR_DTYPE)]),
    # kc, vc, ks, vs, src, dst, n, n_kv, d, page, pages, stream
    *_calls("mx_kv8_copy_pages", [P] * 6 + [3, 2, 64, 16, 9, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in range(6)], *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(6, 11)],
        ({8: 32}, _lib.MX_ERR_SHAPE), ({9: 24}, _lib.MX_ERR_SHAPE), ({0: U}, _lib.MX_ERR_ALIGN), ({3: V}, _lib.MX_ERR_ALIGN),
        ({6: 2 ** 31 - 1}, _lib.MX_ERR_SHAPE), ({7: 2 ** 21, 9: 128, 10: 9}, _lib.MX_ERR_SHAPE)]),
    # q, kc, vc, ks, vs, table, lens, cu, O, B, T, max_q, max_kv, n_q, n_kv, d, page, pages, max_pages, ldq, scale, causal,
    # dtype, workspace, bytes, stream
    *_calls("mx_gqa_kv8", [P] * 9 + [2, 5, 4, 4096, 4, 2, 64, 16, 9, 300, 256, 0.1, 1, 0, P, 1 << 30, None], [
        *[({i: None}, _lib.MX_ERR_NULL) for i in (0, 1, 2, 3, 4, 5, 6, 8)], ({7: None}, _lib.MX_ERR_SHAPE),
        *[({i: 0}, _lib.MX_ERR_SHAPE) for i in range(9, 19)], ({13: 5}, _lib.MX_ERR_SHAPE), ({15: 256}, _lib.MX_ERR_SHAPE),
        ({16: 8}, _lib.MX_ERR_SHAPE), ({19: 248}, _lib.MX_ERR_SHAPE), ({19: 260}, _lib.MX_ERR_ALIGN),
        ({0: U}, _lib.MX_ERR_ALIGN), ({8: U}, _lib.MX_ERR_ALIGN), ({2: U}, _lib.MX_ERR_ALIGN), ({23: U}, _lib.MX_ERR_ALIGN),
        ({22: 2}, _lib.MX_ERR_DTYPE), ({23: None}, _lib.MX_ERR_WORKSPACE), ({24: 1000}, _lib.MX_ERR_WORKSPACE),
        ({10: 2 ** 30}, _lib.MX_ERR_SHAPE), ({18: 2 ** 26 + 1}, _lib.MX_ERR_SHAPE), ({9: 2 ** 22}, _lib.MX_ERR_SHAPE)]),
]


@pytest.mark.parametrize("name,args,code", BAD)
def test_entry_points_refuse(name, args, code):
    assert getattr(_lib.load(), name)(*args) == code


def test_workspaces():
    lib = _lib.load()
    assert lib.mx_linear_int8_workspace(30, 48) == 1536 + 120
    for m, k in ((1, 8192), (2, 4096), (3, 1360), (8, 512), (5, 16)):  # one kernel
        assert lib.mx_linear_int8_workspace(m, k) == 0
    for m, k in ((1, 8208), (2, 4112), (3, 1376), (8, 528), (9, 16)):
        assert lib.mx_linear_int8_workspace(m, k) >= m * (k + 4)
    assert [lib.mx_linear_int8_workspace(*a) for a in ((0, 48), (3, 0), (3, 40), (-1, 16))] == [0] * 4
    assert lib.mx_gqa_kv8_workspace(64, 64, 1, 64, 32, 8, 128) == 0  # one short chunk: no partial results
    assert lib.mx_gqa_kv8_workspace(1, 1, 1, 100000, 32, 8, 128) > 0
    assert lib.mx_gqa_kv8_workspace(1, 1, 1, 100000, 31, 8, 128) == 0


def test_launches_choose(tmp_path):
    """The GPU tests reach every variant of the product; the attention's kernel, its splits and its chunks over many
    sizes: no split starts behind the last token, up to 32 rows per KV head never take the tiles."""
    from test_gpu_int8 import VARIANTS
    sizes = ", ".join(f"{{{v}, {m}, {n}, {k}}}" for v, m, n, k in VARIANTS)
    out = query(tmp_path, "gemm_int8.hip", r"""
  using namespace mx::gemmi8;
  const int sizes[][4] = {SIZES};
  for (auto& s : sizes) printf("%d\n", pick(s[1], s[2], s[3]) == s[0] ? s[0] : -1);
  printf("%d\n", kNumVariants);""".replace("SIZES", sizes))
    assert set(out[:-1]) == {str(v) for v in range(int(out[-1]))}
    out = query(tmp_path, "kv8_attn.hip", r"""
  using namespace mx::kv8;
  long long n = 0;
  for (int B : {1, 3, 64, 4096})
    for (int T : {1, 16, 17, 32, 33, 1000, 100000})
      for (int kv : {1, 255, 256, 257, 8192, 131072, 1 << 30})
        for (int n_kv : {1, 8, 32})
          for (int G : {1, 4, 16, 48})
            for (int max_q : {1, T}) {
              const Plan p = plan(B, T, max_q, kv, n_kv * G, n_kv, T % 2 ? 64 : 128);
              const long long rows = (long long)std::min(max_q, T) * G;
              const bool kernel = rows <= 16 ? p.nr == 1 : rows <= 32 ? p.nr == 2 : p.nr == 0;
              const bool whole = p.splits >= 1 && p.splits <= 65535 && p.chunk >= 1 && p.tiles >= 1;
              const bool useful = p.splits == 1 || (long long)(p.splits - 1) * p.chunk < kv;
              if (!kernel || !whole || !useful) {
                printf("plan(%d, %d, %d, %d, %d, %d)\n", B, T, max_q, kv, n_kv * G, n_kv);
                return 0;
              }
              ++n;
            }
  printf("ok %d\n", n > 1000);""")
    assert out == ["ok 1"]


def test_operators_refuse_before_the_device():
    """Types, shapes and devices that the operators check by themselves: CPU tensors reach no kernel."""
    ops = import_submodule("ops")
    x, w, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for call in (lambda: ops.quant_int8(x), lambda: ops.linear_int8(x, w, s), lambda: ops.gemm_int8(w, s, w, s),
                 lambda: ops.KV8Cache.empty(2, 1, 64, device="cpu")):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    for call in (lambda: ops.quant_int8(x.float()), lambda: ops.linear_int8(x.float(), w, s),
                 lambda: ops.gemm_int8(x, s, w, s), lambda: ops.KV8Cache(x, x, s, s), lambda: ops.quant_int8([1]),
                 lambda: ops.kv8_append(x, x, None, s, s), lambda: ops.gqa_kv8(x, None, s, s),
                 lambda: ops.kv8_copy_pages(None, s, s)):
        with pytest.raises(TypeError):
            call()


def test_numbers_from_the_device_stay_in_bounds(tmp_path):
    """Lengths, row ranges and page numbers of any value: what the kernels make of them."""
    out = query(tmp_path, "kv8_common.h", r"""
  using namespace mx::kv8;
  const int odd[] = {0, 1, 2, 15, 16, 17, 63, 64, 1000, 2147483647, -1, -2, -2147483647 - 1, 1 << 30};
  long long checked = 0;
  for (int lp = 4; lp <= 7; ++lp)
    for (int most : {1, 2, 3, 1 << 24, 2147483647})
      for (int len : odd) {
        const int c = cut_len(len, most, lp);
        if (c < 0 || (long long)c > ((long long)most << lp) || (len >= 0 && (long long)len <= ((long long)most << lp) && c != len)) {
          printf("cut_len(%d, %d, %d) = %d\n", len, most, lp, c);
          return 0;
        }
        ++checked;
      }
  for (int a : odd)
    for (int b : odd)
      for (int T : {1, 5, 64, 2147483647}) {
        const Rows r = cut_rows(a, b, T);
        const bool ok = 0 <= r.first && r.first <= r.last && r.last <= T && (!(0 <= a && a <= b && b <= T) || (r.first == a && r.last == b));
        if (!ok) { printf("cut_rows(%d, %d, %d) = %d, %d\n", a, b, T, r.first, r.last); return 0; }
        ++checked;
      }
  const int row[5] = {3, -1, 9, 10, 0};  // page 10 is none of 10
  for (int lp = 4; lp <= 7; ++lp)
    for (int t : odd) {
      const int p = page_of(row, t, lp, 5, 10);
      const int j = t < 0 ? -1 : t >> lp;
      const int want = j < 0 || j >= 5 || row[j] < 0 || row[j] >= 10 ? -1 : row[j];
      if (p != want) { printf("page_of(%d, %d) = %d\n", t, lp, p); return 0; }
      ++checked;
    }
  printf("ok %d\n", checked > 900);""")
    assert out == ["ok 1"]


# ---- page bookkeeping ------------------------------------------------------
def test_pages_against_a_model():
    """Random extends, forks, truncations, ends and compactions against a model that writes each token into its
    page's slot: every sequence keeps reading what was written for it."""
    for seed in range(30):
        rng = random.Random(seed)
        page = rng.choice([1, 4, 16])
        pool = kv_pages.KVPages(rng.randint(3, 40), page)
        memory = [[None] * page for _ in range(pool.pages)]
        truth, stamp = {}, 0
        for _ in range(300):
            what = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
            if what == "new" or not truth:
                truth[pool.new()] = []
            elif what == "compact":
                moves = pool.compact()
                assert not {a for a, _ in moves} & {b for _, b in moves}
                for a, b in moves:
                    memory[b] = list(memory[a])
                assert sorted({p for s in truth for p in pool.pages_of(s)}) == list(range(pool.pages - pool.free_pages))
            else:
                s = rng.choice(list(truth))
                if what == "fork":
                    truth[pool.fork(s)] = list(truth[s])
                elif what == "free":
                    pool.free(s)
                    del truth[s]
                elif what == "truncate":
                    n = rng.randint(0, len(truth[s]))
                    pool.truncate(s, n)
                    del truth[s][n:]
                else:
                    n = rng.randint(0, 2 * page + 1)
                    before = (pool.pages_of(s), pool.length(s), pool.free_pages)
                    try:
                        copies = pool.extend(s, n)
                    except MemoryError:
                        assert before == (pool.pages_of(s), pool.length(s), pool.free_pages)
                        continue
                    for a, b in copies:
                        memory[b] = list(memory[a])
                    for t in range(len(truth[s]), len(truth[s]) + n):
                        stamp += 1
                        memory[pool.pages_of(s)[t // page]][t % page] = stamp
                        truth[s].append(stamp)
            for s, tokens in truth.items():
                assert pool.length(s) == len(tokens)
                assert [memory[pool.pages_of(s)[t // page]][t % page] for t in range(len(tokens))] == tokens
            assert pool.free_pages + len({p for s in truth for p in pool.pages_of(s)}) == pool.pages


def test_pages_refuse():
    pool = kv_pages.KVPages(2, 16)
    s = pool.new()
    for call, error in ((lambda: pool.extend(9, 1), KeyError), (lambda: pool.fork(9), KeyError), (lambda: pool.free(9), KeyError),
                        (lambda: pool.extend(s, -1), ValueError), (lambda: pool.extend(s, 33), MemoryError),
                        (lambda: pool.truncate(s, 1), ValueError), (lambda: kv_pages.KVPages(0, 16), ValueError),
                        (lambda: pool.table([9]), KeyError)):
        with pytest.raises(error):
            call()
    pool.extend(s, 17)
    with pytest.raises(ValueError):
        pool.table([s], columns=1)
    table, lens = pool.table([s, pool.new()], columns=3)
    assert table.tolist() == [[0, 1, -1], [-1, -1, -1]] and lens.tolist() == [17, 0]
    src, dst = kv_pages.copy_lists([], device="cpu")
    assert src.shape == dst.shape == (0,) and src.dtype == torch.int32


def test_pages_of_a_whole_step_or_of_none():
    """extend_all(): where a later sequence of a step finds no page, the ones before it keep theirs, so that no copy is
    lost; a shared last page is split once for each of its users but one; a sequence may be named twice."""
    pool = kv_pages.KVPages(3, 16)
    a = pool.new()
    pool.extend(a, 20)
    c = pool.fork(a)
    before = [(pool.pages_of(s), pool.length(s)) for s in (a, c)]
    with pytest.raises(MemoryError):
        pool.extend_all([(a, 1), (c, 14)])
    with pytest.raises(KeyError):
        pool.extend_all([(a, 1), (9, 1)])
    with pytest.raises(ValueError):
        pool.extend_all([(a, 1), (c, -1)])
    assert before == [(pool.pages_of(s), pool.length(s)) for s in (a, c)] and pool.free_pages == 1
    assert pool.extend_all(iter([(a, 1), (c, 12)])) == [(1, 2)]
    assert (pool.pages_of(a), pool.pages_of(c)) == ((0, 2), (0, 1))
    assert pool.extend_all([]) == pool.extend_all([(a, 0)]) == []

    pool = kv_pages.KVPages(9, 16)
    a = pool.new()
    pool.extend(a, 5)
    forks = [a] + [pool.fork(a) for _ in range(3)]
    assert pool.extend_all([(s, 1) for s in forks]) == [(0, 1), (0, 2), (0, 3)]
    assert [pool.pages_of(s) for s in forks] == [(1,), (2,), (3,), (0,)]
    d = pool.fork(a)
    assert pool.extend_all([(d, 10), (d, 3)]) == [(1, 4)]
    assert pool.pages_of(d) == (4, 5) and pool.length(d) == 19 and pool.pages_of(a) == (1,)


def test_pages_of_steps_against_a_model():
    """Random steps of several sequences, forks and ends, in pools that are often full: a step that fails changes
    nothing, one that succeeds gives copies whose targets are new, and what was written stays readable."""
    failed = 0
    for seed in range(40):
        rng = random.Random(seed)
        page = rng.choice([1, 4, 16])
        pool = kv_pages.KVPages(rng.randint(2, 14), page)
        memory = [[None] * page for _ in range(pool.pages)]
        truth, stamp = {}, 0
        for _ in range(150):
            what = rng.choice(["new", "step", "step", "step", "fork", "free"])
            if what == "new" or not truth:
                truth[pool.new()] = []
            elif what == "fork":
                s = rng.choice(list(truth))
                truth[pool.fork(s)] = list(truth[s])
            elif what == "free":
                s = rng.choice(list(truth))
                pool.free(s)
                del truth[s]
            else:
                step = [(rng.choice(list(truth)), rng.randint(0, page + 1)) for _ in range(rng.randint(1, 5))]
                before = ({s: (pool.pages_of(s), pool.length(s)) for s in truth}, pool.free_pages)
                used = {p for s in truth for p in pool.pages_of(s)}
                try:
                    copies = pool.extend_all(step)
                except MemoryError:
                    failed += 1
                    assert before == ({s: (pool.pages_of(s), pool.length(s)) for s in truth}, pool.free_pages)
                    continue
                targets = [b for _, b in copies]
                assert len(set(targets)) == len(targets) and not set(targets) & used
                for a, b in copies:
                    memory[b] = list(memory[a])
                for s, n in step:
                    for _ in range(n):
                        stamp += 1
                        t = len(truth[s])
                        memory[pool.pages_of(s)[t // page]][t % page] = stamp
                        truth[s].append(stamp)
            for s, tokens in truth.items():
                assert pool.length(s) == len(tokens)
                assert [memory[pool.pages_of(s)[t // page]][t % page] for t in range(len(tokens))] == tokens
    assert failed > 100


def test_pages_take_whole_numbers_of_tokens():
    """A count that is no whole number is refused before anything has changed; numpy's and torch's integers count."""
    pool = kv_pages.KVPages(6, 16)
    a = pool.new()
    pool.extend(a, 20)
    c = pool.fork(a)
    for tokens in (17.0, float("nan"), "3", None, torch.tensor(2.0)):
        with pytest.raises(TypeError):
            pool.extend(c, tokens)
    assert pool.pages_of(c) == pool.pages_of(a) == (0, 1) and pool.length(c) == 20 and pool.free_pages == 4
    assert pool.extend(c, torch.tensor([3, 17], dtype=torch.int32)[1]) == [(1, 2)]
    assert pool.length(c) == 37 and type(pool.length(c)) is int


def test_split_launches_cover_each_kernel(tmp_path):
    """The cases of test_attend_split: each kernel (16 rows, 32 rows, tiles) with pages of less than 64 tokens and of
    more, at d = 64 and 128, has its keys split in one at least."""
    from test_gpu_kv8_edges import SPLIT
    sizes = ", ".join("{%d, %d, %d, %d, %d, %d}" % (len(lens), sum(news), max(news), -(-max(lens) // page) * page, n_kv * group, n_kv)
                      for d, page, n_kv, group, lens, news in SPLIT)
    ds = ", ".join(str(case[0]) for case in SPLIT)
    out = query(tmp_path, "kv8_attn.hip", r"""
  using namespace mx::kv8;
  const int s[][6] = {SIZES}, ds[] = {DS};
  int i = 0;
  for (auto& c : s) {
    const Plan p = plan(c[0], c[1], c[2], c[3], c[4], c[5], ds[i++]);
    printf("%d %d\n", p.nr, p.splits > 1);
  }""".replace("SIZES", sizes).replace("DS", ds))
    got = {(line.split()[0], case[1] >= 64, case[0]) for line, case in zip(out, SPLIT) if line.endswith(" 1")}
    assert got == {(nr, wide, d) for nr in "120" for wide in (False, True) for d in (64, 128)}, out
