"""The 8-bit cache and the page copies without a GPU: the kernels' integer arithmetic, the C structs, what is refused."""
import ctypes as C
import os
import re
import subprocess
import types

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run_c(tmp_path, source, compiler="g++", name="t"):
    src = tmp_path / f"{name}.{'c' if compiler == 'gcc' else 'cpp'}"
    src.write_text(source)
    exe = tmp_path / name
    subprocess.run([compiler, "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "bi-kv_amd", "csrc"), str(src), "-o", str(exe), "-lpthread"], check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()


def test_division_without_dividing_is_exact(tmp_path):
    """Every divisor up to 65536 (tokens of a page) at the quotient's steps and the range's ends."""
    out = _run_c(tmp_path, r"""
#include <stdio.h>
#include <initializer_list>
#include "host_logic/fp8_logic.h"
int main() {
  const uint32_t top = 0x7fffffffu;
  long bad = 0, n = 0;
  for (uint32_t d = 1; d <= 65536; ++d) {
    const bikv::FastDiv f = bikv::fast_div(d);
    for (uint32_t k : {0u, 1u, 2u, top / d / 2, top / d - (top / d > 0), top / d})
      for (int64_t x : {(int64_t)k * d - 1, (int64_t)k * d, (int64_t)k * d + 1})
        if (x >= 0 && x <= top) { ++n; bad += bikv::divide((uint32_t)x, f) != (uint32_t)x / d; }
    for (uint32_t x : {top, top - 1, top - d}) { ++n; bad += bikv::divide(x, f) != x / d; }
  }
  for (uint32_t d : {65537u, 99991u, 1u << 20, 0x3fffffffu, 0x40000000u, 0x40000001u, top}) {
    const bikv::FastDiv f = bikv::fast_div(d);
    for (uint32_t x : {0u, 1u, d - 1, d, top - 1, top}) { ++n; bad += bikv::divide(x, f) != x / d; }
  }
  printf("%ld %ld\n", bad, n);
}
""")
    assert out[0] == "0" and int(out[1]) > 1000000


def test_shares_cover_the_work_once_and_in_order(tmp_path):
    """Shares are adjacent, end where the work ends, and step x lies in share x / per, also near 2^31 steps."""
    out = _run_c(tmp_path, r"""
#include <stdio.h>
#include <initializer_list>
#include "host_logic/fp8_logic.h"
int main() {
  long bad = 0;
  for (uint32_t total : {0u, 1u, 7u, 8u, 255u, 256u, 257u, 5000u, 1u << 20, 0x7ffffff0u, 0x7fffffffu})
    for (uint32_t slots : {1u, 2u, 32u, 51u, 85u, 256u})
      for (uint32_t least : {1u, 2u, 8u}) {
        uint32_t at = 0;
        for (uint32_t s = 0; s < slots; ++s) {
          const bikv::Share h = bikv::share_of(total, slots, least, s);
          bad += h.begin != at || h.end < h.begin || h.end > total;
          if (h.begin < h.end) {
            bad += h.begin / h.per != s || (h.end - 1) / h.per != s;
            bad += h.end != total && h.end - h.begin < least;
          }
          at = h.end;
        }
        bad += at != total;
      }
  printf("%ld\n", bad);
}
""")
    assert out == ["0"]


def test_the_line_of_few_rows_work_stays_below_2_31(tmp_path):
    """Every tile's key steps and what beginning it costs, for as many tiles as a call may have: signed 32-bit numbers count them."""
    out = _run_c(tmp_path, r"""
#include <stdio.h>
#include <initializer_list>
#include "host_logic/attend_plan.h"
int main() {
  long bad = 0, few = 0, n = 0, close = 0;
  for (int heads : {1, 2, 3, 5, 8, 9, 1024})
    for (int group : {1, 4, 7, 16, 32})
      for (int one_each : {0, 1})
        for (int64_t seqs : {int64_t(1), int64_t(9), int64_t(1000), int64_t(1) << 20, (int64_t(1) << 24) - 1})
          for (int64_t rows_each : {1, 2, 4, 8, 16, 31})
            for (int64_t len = 0; len <= (int64_t(1) << 30); len = len < 4096 ? len + 32 : len * 2 + 1) {
              const int64_t rows = one_each ? seqs : seqs * rows_each;
              if (rows >= (int64_t(1) << 30)) continue;
              const bikv::AttendPlan p = bikv::plan_fp8_attend(heads, group, one_each, seqs, rows, len);
              ++n;
              if (p.form == bikv::ATTEND_MANY) continue;
              const int64_t line = p.tiles * (bikv::steps_of_keys(len, p.form == bikv::ATTEND_FEW_16 ? 64 : 32) + p.begin_cost);
              ++few;
              bad += line >= (int64_t(1) << 31);
              close += line > (int64_t(1) << 31) / 10 * 9;
            }
  printf("%ld %ld %ld %ld\n", bad, few, n, close);
}
""")
    assert out[0] == "0" and int(out[1]) > 10000 and int(out[3]) > 5


def test_launches_of_more_threads_than_a_launch_numbers_do_not_fit(tmp_path):
    out = _run_c(tmp_path, r"""
#include <stdio.h>
#include "host_logic/attend_plan.h"
#include "host_logic/fp8_logic.h"
using namespace bikv;
static int attend(int heads, int group, bool one_each, int64_t seqs, int64_t rows, int64_t len) {
  const AttendPlan p = plan_fp8_attend(heads, group, one_each, seqs, rows, len);
  const bool fits = launch_fits(p.groups, p.threads);
  return fits == (p.groups * p.threads < (int64_t(1) << 32)) ? fits : -1;
}
static int append(int heads, bool one_each, int64_t seqs, int64_t rows, int page) {
  const int64_t groups = append_groups(append_units(one_each, seqs, rows, page), heads);
  return launch_fits(groups, kAppendThreads) == (groups * kAppendThreads < (int64_t(1) << 32)) ? launch_fits(groups, kAppendThreads) : -1;
}
int main() {
  printf("%d%d%d%d ", launch_fits((int64_t(1) << 24) - 1, 256), launch_fits(int64_t(1) << 24, 256), launch_fits((int64_t(1) << 23) - 1, 512), launch_fits(int64_t(1) << 23, 512));
  printf("%d%d%d%d ", append(64, false, 1, 600000, 1), append(64, false, 1, 500000, 1), append(8, true, 4000000, 4000000, 16), append(8, true, 1 << 23, 1 << 23, 16));
  printf("%d%d%d%d ", attend(9, 1, true, 5000000, 5000000, 1000), attend(9, 1, true, 4000000, 4000000, 1000), attend(9, 1, true, 5000000, 5000000, 2000), attend(8, 1, false, 8, 1 << 29, 4096));
  printf("%d\n", attend(1024, 4, false, 1 << 20, 1 << 24, 64));
}
""")
    # the last five: 5 and 4 million workgroup pairs of 512 threads; shares, which are few whatever the call; 2^22 tiles of 8 heads; 2^20 of 1024
    assert out == ["1010", "0110", "0110", "0"]


def test_assembly_that_writes_m0_says_so():
    """The compiler keeps values of its own in m0."""
    csrc = os.path.join(ROOT, "bi-kv_amd", "csrc")
    found = 0
    for name in sorted(os.listdir(csrc)):
        if name.endswith((".hip", ".h")):
            with open(os.path.join(csrc, name)) as f:
                text = f.read()
            for stmt in re.findall(r"\basm\b[^;]*;", text):
                if re.search(r"\bs_mov_b32 m0\b", stmt):
                    found += 1
                    assert '"m0")' in stmt, (name, stmt)
    assert found >= 2


def test_lds_that_is_read_four_floats_at_a_time_is_aligned_for_it():
    """A struct without a 16-byte member is where the compiler likes to put it, unless it says what it needs."""
    with open(os.path.join(ROOT, "bi-kv_amd", "csrc", "fp8_cache_attend.hip")) as f:
        structs = re.findall(r"struct (alignas\(16\) )?Meta \{(.*?)\n  \};(.*?)\n  __shared__", f.read(), re.S)
    assert len(structs) == 2
    for aligned, members, after in structs:
        assert aligned or "u32x4" in members
        assert all(f"offsetof(Meta, {m}) % 16 == 0" in after for m in ("ks", "vs", "ex"))


def test_structs_agree_with_the_header(lib, tmp_path):
    from bikv_pagecopy import _lib, fp8_cache
    fields = [n for n, _ in _lib.FP8CacheDesc._fields_]
    batch = ["page_table", "page_table_stride", "max_pages", "kv_lens", "q_starts", "n_seqs", "n_rows", "dtype", "reserved"]
    out = _run_c(tmp_path, "#include <stddef.h>\n#include <stdio.h>\n#include \"bikv_pagecopy.h\"\nint main(void) {\n"
                 + "".join(f'  printf("%zu\\n", offsetof(bikv_fp8_cache_desc, {f}));\n' for f in fields)
                 + "".join(f'  printf("%zu\\n", offsetof(bikv_seq_batch, {f}));\n' for f in batch)
                 + '  printf("%zu %zu %d %d\\n", sizeof(bikv_fp8_cache_desc), sizeof(bikv_seq_batch), BIKV_T_BF16, BIKV_T_FP16);\n  return 0;\n}\n', "gcc")
    want = [getattr(_lib.FP8CacheDesc, f).offset for f in fields] + [0, 8, 16, 24, 32, 40, 48, 56, 60]
    assert [int(x) for x in out] == want + [C.sizeof(_lib.FP8CacheDesc), fp8_cache._SEQ_BATCH.size, _lib.T_BF16, _lib.T_FP16]


def _desc(**change):
    from bikv_pagecopy import _lib
    d = _lib.FP8CacheDesc()
    d.device, d.n_layers, d.kv_heads, d.head_dim, d.page_tokens, d.n_pages = 0, 1, 2, 128, 16, 4
    d.token_stride_bytes, d.page_stride_bytes, d.scale_page_stride_bytes = 256, 4096, 8
    d.planes = (C.c_void_p * 2)(4096, 8192)                  # addresses that nothing here looks at
    d.scales = (C.c_void_p * 2)(4096, 8192)
    for name, value in change.items():
        if name == "planes":
            d.planes[1] = value
        elif name == "scales":
            d.scales[1] = value
        else:
            setattr(d, name, value)
    if "plane_base" not in change:
        d.plane_base = C.cast(d.planes, C.POINTER(C.c_void_p))
    if "scale_plane_base" not in change:
        d.scale_plane_base = C.cast(d.scales, C.POINTER(C.c_void_p))
    return d


@pytest.mark.parametrize("change", [
    dict(n_layers=0), dict(n_layers=-1), dict(n_layers=1 << 20), dict(kv_heads=0), dict(kv_heads=1025), dict(head_dim=0), dict(head_dim=96), dict(head_dim=256),
    dict(page_tokens=0), dict(page_tokens=65537), dict(n_pages=0), dict(n_pages=-3), dict(n_pages=1 << 61), dict(token_stride_bytes=128), dict(token_stride_bytes=264),
    dict(token_stride_bytes=1 << 31), dict(page_stride_bytes=4080), dict(page_stride_bytes=4104), dict(scale_page_stride_bytes=4), dict(scale_page_stride_bytes=10),
    dict(plane_base=None), dict(scale_plane_base=None), dict(planes=None), dict(planes=4104), dict(scales=None), dict(scales=4098)], ids=str)
def test_a_cache_that_makes_no_sense_is_refused(lib, change):
    from bikv_pagecopy import _lib
    h = C.c_void_p()
    assert lib.bikv_fp8_cache_create(C.byref(_desc(**change)), C.byref(h)) == _lib.EINVAL
    assert not h.value and _lib.last_error()


def test_null_arguments_are_refused(lib):
    from bikv_pagecopy import _lib
    h = C.c_void_p()
    assert lib.bikv_fp8_cache_create(None, C.byref(h)) == _lib.EINVAL
    assert lib.bikv_fp8_cache_create(C.byref(_desc()), None) == _lib.EINVAL
    assert lib.bikv_fp8_cache_destroy(None) == _lib.OK
    assert lib.bikv_fp8_append(None, 0, None, None, 0, 0, None, 0, 0, None) == _lib.EINVAL
    assert lib.bikv_fp8_attend(None, 0, None, None, 0, 0, 1, 1, 1.0, None, 0, 0, None, None, 0, None) == _lib.EINVAL
    assert lib.bikv_fp8_attend_workspace(None, None, 1) == _lib.EINVAL
    assert lib.bikv_copy_pages(None, None, None, 0, None) == _lib.EINVAL


# ---- the Python layer's own checks, over tensors of the host -------------------------------------
def _bare(heads=2, dim=128):
    from bikv_pagecopy import FP8KVCache
    c = FP8KVCache.__new__(FP8KVCache)
    c._h, c.pool, c.device, c.kv_heads, c.head_dim = None, None, torch.device("cpu"), heads, dim
    return c


def test_rows_that_the_kernels_cannot_read_are_refused(lib):
    c = _bare()
    ok = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    assert c._rows("k", ok, 2) == (256, 128, 1)
    assert c._rows("k", torch.zeros(3, 4, 256, dtype=torch.float16)[:, 1:3, 128:], 2) == (1024, 256, 1)
    for bad, heads in ((ok.float(), 2), (ok, 3), (ok[..., :64], 2), (ok[0], 2), (ok.transpose(0, 2).contiguous().transpose(0, 2), 2), (ok.to("meta"), 2)):
        with pytest.raises(RuntimeError, match="k"):
            c._rows("k", bad, heads)
    wants = ok.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="gradient"):
        c._rows("q", wants, None)
    with torch.no_grad():
        c._rows("q", wants, None)


def test_tensors_with_a_forward_mode_gradient_are_refused(lib):
    """A tangent would be lost without a word, under no_grad too, which turns off the other mode only."""
    import torch.autograd.forward_ad as fa
    c = _bare()
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with fa.dual_level():
        dual = fa.make_dual(x, torch.ones_like(x))
        for t in (dual, dual[1:], dual[:, :1]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                c._rows("q", t, None)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                c._rows("q", t, None)
        c._rows("q", x, None)
        c._rows("q", fa.unpack_dual(dual).primal, None)
    c._rows("q", dual, None)                                 # the level is gone, and the tangent with it


def test_a_cache_over_tensors_that_want_a_gradient_is_refused(lib):
    """Attention over a scale that is learnt would leave it without a gradient."""
    import torch.autograd.forward_ad as fa
    from bikv_pagecopy import FP8KVCache
    scale = torch.ones(3, 2)
    for wants in ([scale, scale.clone().requires_grad_()], [torch.nn.Parameter(scale)]):
        with pytest.raises(RuntimeError, match="gradient"):
            FP8KVCache._refuse_gradients(wants)
        with torch.no_grad():
            FP8KVCache._refuse_gradients(wants)
    FP8KVCache._refuse_gradients([scale])
    with fa.dual_level(), pytest.raises(RuntimeError, match="gradient"):
        FP8KVCache._refuse_gradients([fa.make_dual(scale, scale)])


def test_sequence_arrays_that_are_not_what_a_call_takes_are_refused(lib):
    c = _bare()
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    table, lens, starts = torch.zeros(2, 5, dtype=torch.int64), torch.ones(2, dtype=torch.int64), torch.tensor([0, 1, 3])
    assert len(c._batch(k, table, lens, starts)) == 64
    assert len(c._batch(k[:2], table[:, :3], lens, None)) == 64
    for t, l, s in ((table.int(), lens, starts), (table, lens.int(), starts), (table, lens, starts.int()), (table[0], lens, starts), (table, lens[:1], starts),
                    (table, lens, starts[:2]), (table, lens, None), (table.t().contiguous().t(), lens, starts), (table[:1].expand(2, 5), lens, starts),
                    (table, torch.ones(4, dtype=torch.int64)[::2], starts), (table, lens, torch.zeros(6, dtype=torch.int64)[::2]),
                    (table.to("meta"), lens, starts), (table, lens.to("meta"), starts), (table, lens, starts.to("meta")), (table, lens[None], starts)):
        with pytest.raises(RuntimeError):
            c._batch(k, t, l, s)


def test_page_moves_that_contradict_each_other_are_refused(lib):
    from bikv_pagecopy import PagedKVPool
    pool = types.SimpleNamespace(n_pages=10, device=torch.device("cpu"))
    for src, dst in (([0, 3, 3], [1, 2, 9]), ([], []), ([4], [4]), ([4, 4], [4, 5]), (np.arange(3), torch.arange(3, 6))):
        s, d = PagedKVPool.page_moves(pool, src, dst)
        assert s.dtype == d.dtype == torch.int64 and s.is_contiguous() and d.is_contiguous()
        assert s.tolist() == list(map(int, src)) and d.tolist() == list(map(int, dst))
    for src, dst in (([0], [1, 2]), ([-1], [1]), ([10], [1]), ([1], [10]), ([1], [-2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0, 1], [1, 0])):
        with pytest.raises(RuntimeError):
            PagedKVPool.page_moves(pool, src, dst)


def test_a_cache_on_the_host_is_refused(lib):
    from bikv_pagecopy import FP8KVCache
    payload, scale = torch.zeros(1, 2, 3, 16, 2, 128, dtype=torch.uint8), torch.ones(1, 2, 3, 2)
    for make in (lambda: FP8KVCache(payload, scale), lambda: FP8KVCache(payload[:, :1], scale), lambda: FP8KVCache(payload, scale[..., :1]), lambda: FP8KVCache.from_planes([], []),
                 lambda: FP8KVCache.from_planes([payload[0, 0], payload[0, 1]], [scale[0, 0], scale[0, 1]])):
        with pytest.raises(RuntimeError):
            make()
