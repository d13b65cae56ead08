"""How linear_xent divides a call (csrc/common/linear_xent_plan.hpp, compiled
here by g++): its scratch, the parts of the classes and the shares of dX."""
from __future__ import annotations

import ctypes
import random
import shutil
import subprocess

import pytest

from test_gemm_codegen import REPO

CODE = """
#include "linear_xent_plan.hpp"
using namespace aicf::hip;
extern "C" int64_t plan(int64_t R, int64_t V, int64_t D, int64_t ldw, int direct, int f32, int grad, int64_t piece,
                        int64_t bytes, int64_t ob, int64_t* out, int64_t* v0, int64_t* cols, int64_t most) {
  LxPlan p;
  if (!lx_plan(R, V, D, ldw, direct, f32, grad, piece, bytes, &p)) return -1;
  if (ob > 0) p.held = lx_held(p, V, D, ldw, ob);
  const LxParts q = lx_parts(p, V, grad);
  const int64_t o[] = {p.Rp, p.Dp, p.piece, p.held, p.slab_rows, p.stats_off, p.xc_off, p.slab_off, p.wpad_off,
                       p.g_off, p.bytes, p.bn, p.bm_dx, q.longest(), q.kept, p.bm};
  std::copy(o, o + sizeof o / 8, out);
  for (int64_t k = 0; k < q.count && k < most; ++k) {
    v0[k] = q.at(k).v0;
    cols[k] = q.at(k).cols;
  }
  return q.count;
}
extern "C" int share_k(int k, int shares) { return lx_share_k(k, shares); }
extern "C" int slabs(int k, int share) { return lx_slabs(k, share); }
"""
NAMES = ("Rp", "Dp", "piece", "held", "slab_rows", "stats_off", "xc_off", "slab_off", "wpad_off", "g_off", "bytes",
         "bn", "bm_dx", "longest", "kept", "bm")
MOST = 4096


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("lx_plan")
    (d / "plan.cpp").write_text(CODE)
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-I{REPO / 'ai-compiler-framework_amd' / 'csrc' / 'common'}", str(d / "plan.cpp"), "-o", str(d / "plan.so")]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    so = ctypes.CDLL(str(d / "plan.so"))
    i64, ptr = ctypes.c_int64, ctypes.POINTER(ctypes.c_int64)
    so.plan.restype, so.plan.argtypes = i64, [i64] * 4 + [ctypes.c_int] * 3 + [i64] * 3 + [ptr] * 3 + [i64]
    return so


def plan(lib, r, v, d, f32=False, grad=True, piece=0, ob=0, direct=None, ldw=None, scratch=-1):
    """(the plan's numbers, its first parts [(first class, classes)]), or None."""
    if direct is None:
        direct = d * (4 if f32 else 2) % 16 == 0
    out, v0, cols = (ctypes.c_int64 * len(NAMES))(), (ctypes.c_int64 * MOST)(), (ctypes.c_int64 * MOST)()
    n = lib.plan(r, v, d, ldw or d, direct, f32, grad, piece, scratch, ob, out, v0, cols, MOST)
    if n < 0:
        return None
    n = min(n, MOST)
    return dict(zip(NAMES, out)), list(zip(v0[:n], cols[:n]))


def check(lib, r, v, d, f32, grad, ob, p, parts):
    es = 4 if f32 else 2
    direct = d * es % 16 == 0
    # every class is in one part, and no part in scratch or dW is longer than its place
    at = 0
    for v0, cols in sorted(parts):
        assert v0 == at and cols > 0
        at += cols
    assert at == v
    assert all(cols <= (p["held"] if p["held"] and k == 0 else p["piece"]) for k, (_, cols) in enumerate(parts))
    # scratch: each array in front of the next
    sizes = [("stats_off", -(-v // 256) * 256 // p["bn"] * p["Rp"] * 8), ("xc_off", p["Rp"] * p["Dp"] * es)]
    if grad:
        sizes += [("slab_off", p["slab_rows"] * p["Dp"] * 4), ("g_off", p["Rp"] * p["piece"] * es)]
    if not direct:
        sizes += [("wpad_off", p["piece"] * p["Dp"] * es)]
    spans = sorted((p[n], p[n] + s) for n, s in sizes)
    assert spans[0][0] >= 256 + 8 * 4 * p["Rp"] and all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    if grad:
        # every slab that is joined is one that the longest part writes, for any number of shares
        longest = max(cols for _, cols in parts)
        for shares in range(1, 65):
            k = lib.share_k(p["longest"], shares)
            joined = lib.slabs(p["longest"], k)
            assert joined <= shares and k % 64 == 0
            assert (joined - 1) * k < longest, (shares, k, joined, longest)
        assert p["longest"] == longest
        if p["held"]:  # G behind the rows of dW that its part writes, on 256 bytes
            assert p["held"] * d * ob + 255 + p["Rp"] * p["held"] * es <= v * d * ob


# parts shorter than the piece that they are given: r, v, d, piece
SHORT = [(128, 5889, 512, 5376), (512, 50257, 768, 49408), (16, 12344, 128, 6400), (1, 10270, 512, 5376),
         (64, 28436, 128, 28416)]


@pytest.mark.parametrize("r,v,d,piece", SHORT)
def test_parts_shorter_than_a_piece(lib, r, v, d, piece):
    for ob in (0, 2, 4):
        p, parts = plan(lib, r, v, d, piece=piece, ob=ob)
        check(lib, r, v, d, False, True, ob, p, parts)
        assert max(c for _, c in parts) < piece


def test_any_sizes(lib):
    rng = random.Random(8)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    seen = 0
    for _ in range(20000):
        r, v, d, f32, grad = log(1, 9000), log(1, 300000), log(1, 9000), rng.random() < 0.3, rng.random() < 0.9
        piece = rng.choice((0, log(1, v), max(1, v - log(1, v)), v))
        if piece and v / piece > 500:
            continue
        ob = rng.choice((0, 2, 4)) if grad else 0
        got = plan(lib, r, v, d, f32, grad, piece, 4 if f32 and ob else ob)
        if got is None:
            assert d * 256 * (4 if f32 else 2) >= 2 ** 31 - 1 or (grad and r * d * 4 > 2 ** 29)
            continue
        check(lib, r, v, d, f32, grad, 4 if f32 and ob else ob, *got)
        p = got[0]
        if rng.random() < 0.2:  # exactly the bytes that it asks for, and more
            again = plan(lib, r, v, d, f32, grad, 0, 4 if f32 and ob else ob, scratch=p["bytes"])
            assert again[0]["piece"] >= p["piece"] and again[0]["bytes"] <= p["bytes"]
            check(lib, r, v, d, f32, grad, 4 if f32 and ob else ob, *again)
            more = plan(lib, r, v, d, f32, grad, 0, 4 if f32 and ob else ob, scratch=p["bytes"] + log(1, 10 ** 9))
            check(lib, r, v, d, f32, grad, 4 if f32 and ob else ob, *more)
        seen += len(got[1]) > 1
    assert seen > 3000


def test_launches_stay_below_2_32_work_items(lib):
    """The largest calls: copies of rows (a wave each) and the logits' tiles, 256 threads each unless workgroups of
    512 loop over them; what would need more is refused, or done in smaller pieces."""
    def launches(r, v, d, f32):
        """Work-items of the copies and tiles of the logits' launch, or None where the call is refused."""
        got = plan(lib, r, v, d, f32, grad=False)
        if got is None:
            return None
        p, parts = got
        direct = d * (4 if f32 else 2) % 16 == 0
        cols = v if direct else max(c for _, c in parts)
        copies = max(r, 0 if direct else cols)
        return -(-copies // 4) * 256, -(-r // p["bm"]) * -(-cols // p["bn"]), p["bm"]

    rng = random.Random(3)
    taken = refused = 0
    for _ in range(4000):
        r, v, d = (int(2 ** rng.uniform(0, top)) for top in (30, 28, 12))
        d = max(1, d // 8 * 8) if rng.random() < 0.7 else d
        f32 = rng.random() < 0.5
        got = launches(r, v, d, f32)
        if got is None:
            refused += 1
            assert r >= 2 ** 26 - 256 or r * v > 2 ** 35
            continue
        copies, tiles, bm = got
        looped = bm == 256 and not f32 and (d if d * 2 % 16 == 0 else -(-d // 64) * 64) < 2048
        assert copies < 2 ** 32 and tiles < (2 ** 31 - 1024 if looped else 2 ** 24)
        taken += 1
    assert taken > 1000 and refused > 100
    assert launches(1, 2 ** 28, 64, False) and launches(2 ** 26 - 256, 1000, 64, False)
    assert launches(2 ** 26, 1000, 64, False) is None
    for f32, d, r, v, ok in ((True, 64, 2 ** 18, 2 ** 17, True), (True, 64, 2 ** 20, 2 ** 20, False),
                             (False, 4096, 2 ** 20, 2 ** 19, True), (False, 4096, 2 ** 20, 2 ** 20, False),
                             (False, 1024, 2 ** 20, 2 ** 20, True), (False, 1024, 2 ** 24, 2 ** 24, False),
                             (True, 65, 2 ** 20, 2 ** 20, True)):  # (rows of W copied: by pieces)
        assert (launches(r, v, d, f32) is not None) == ok, (f32, d, r, v)
