"""How expert_linear's tensor-core kernel cuts its work: the functions of csrc/tokens.cu, compiled for the host as they stand there.  Every
token of every segment and every block of channels comes in exactly one tile, a tile's columns are a multiple of 16 that the boxes
cover without leaving the tile's shared memory, and the division by multiplication is exact over its range."""
import ctypes
import os
import random
import re
import subprocess

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_int8_b200", "csrc", "tokens.cu")

HEAD = r"""
#include <stdint.h>
#define __device__
#define __forceinline__ inline
#define __align__(n) alignas(n)
static uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }
static int __clz(int v) { return v ? __builtin_clz((unsigned)v) : 32; }
struct TokenArgs { int experts; };
struct GroupArgs { TokenArgs t; int n_tiles, cap; uint32_t by_cap; };
"""
TAIL = r"""
static uint32_t by[RASTER + 1];
static void init() { for (uint32_t w = 2; w <= RASTER; ++w) by[w] = 0xffffffffu / w + 1; }
static int cut(const GroupArgs& p, const int* rows, int experts, int n_tiles, Segment* seg) {
  init();
  int at = 0, first = 0;
  for (int e = 0; e < experts; ++e) {
    const int count = rows[e], tiles = tiles_of(count, p);
    seg[e].row = at; seg[e].rows = count;
    seg[e].share = tiles ? ((count + tiles - 1) / tiles + 15) & ~15 : 0;
    seg[e].first = first;
    at += count; first += tiles * n_tiles;
  }
  seg[experts].first = first;
  return first;
}
extern "C" int tiles(int tok, int cap, const int* rows, int experts, int n_tiles, int* out) {   // out: expert, channel, row, rows, columns, loaded
  static Segment seg[2048];
  const GroupArgs p{{experts}, n_tiles, cap / 16, 0xffffffffu / (cap / 16) + 1};
  const int total = cut(p, rows, experts, n_tiles, seg);
  for (int t = 0; out && t < total; ++t, out += 6) {
    const Tile r = tok == 64 ? tile_of<64>(t, p, seg, by) : tok == 128 ? tile_of<128>(t, p, seg, by) : tile_of<256>(t, p, seg, by);
    out[0] = r.expert; out[1] = r.channel; out[2] = (int)r.row; out[3] = r.rows; out[4] = r.columns; out[5] = boxes_of(r.columns).tokens();
  }
  return total;
}
extern "C" int quotient(uint32_t n, int w) { init(); return (int)__umulhi(n, by[w]); }
"""


def _take(text, pattern):
    return re.search(pattern, text, re.S | re.M).group(0)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    text = open(SRC).read()
    parts = [_take(text, r"^constexpr int GRP_THREADS = [^;]*;"), _take(text, r"^constexpr int RASTER = [^;]*;"),
             _take(text, r"^struct __align__\(16\) Segment \{.*?^\};"), _take(text, r"^struct Tile \{.*?^\};"),
             _take(text, r"^struct Boxes \{.*?^\};"), _take(text, r"^__device__ __forceinline__ Boxes boxes_of.*?^\}"),
             _take(text, r"^__device__ __forceinline__ int tiles_of.*?\}$"),
             _take(text, r"^template <int TOK>\n__device__ __forceinline__ Tile tile_of.*?^\}")]
    tmp = tmp_path_factory.mktemp("tiles")
    src, so = tmp / "tiles.cpp", tmp / "tiles.so"
    src.write_text(HEAD + "\n".join(parts) + TAIL)
    subprocess.run([os.environ.get("CXX") or "g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-o", str(so), str(src)], check=True)
    return ctypes.CDLL(str(so))


@pytest.mark.parametrize("tok, cap", [(64, 64), (128, 128), (256, 256), (128, 80), (128, 96), (256, 144), (256, 240)])
def test_every_token_and_channel_once(lib, tok, cap):
    rng = random.Random(cap)
    cases = [[1], [16], [17], [63, 64, 65], [0, 0, 5, 0], [0], [255, 256, 257, 0, 1], [4096], [4097], [cap * 16], [cap * 16 + 1], [9000, 3], [1] * 300]
    cases += [[rng.choice([0, 1, 7, rng.randrange(2000)]) for _ in range(rng.randrange(1, 40))] for _ in range(20)]
    for rows in cases:
        for n_tiles in (1, 3, 17):
            arr = (ctypes.c_int * len(rows))(*rows)
            total = lib.tiles(tok, cap, arr, len(rows), n_tiles, None)
            assert total == sum(-(-r // cap) for r in rows) * n_tiles
            assert total <= (sum(rows) // cap + sum(1 for r in rows if r)) * n_tiles   # what the host reckons with
            out = (ctypes.c_int * max(1, 6 * total))()
            lib.tiles(tok, cap, arr, len(rows), n_tiles, out)
            begin = [sum(rows[:e]) for e in range(len(rows))]
            seen = {}
            for t in range(total):
                e, channel, row, count, columns, loaded = out[6 * t:6 * t + 6]
                assert 0 < count <= columns <= cap and columns % 16 == 0 and columns - count < 16
                assert columns <= loaded <= tok and channel % 128 == 0 and 0 <= channel < 128 * n_tiles
                assert begin[e] <= row and row + count <= begin[e] + rows[e]
                seen.setdefault((e, channel), []).append((row, row + count))
            for e, r in enumerate(rows):
                for n in range(n_tiles):
                    spans = sorted(seen.get((e, 128 * n), []))
                    assert sum(b - a for a, b in spans) == r
                    assert all(x[1] == y[0] for x, y in zip(spans, spans[1:])) and (not r or spans[0][0] == begin[e])


def test_division_by_multiplication(lib):
    rng = random.Random(1)
    lib.quotient.argtypes = [ctypes.c_uint32, ctypes.c_int]
    for w in range(2, 17):
        for n in [*range(200), (1 << 28) - 1, (1 << 28) - w, *(rng.randrange(1 << 28) for _ in range(2000)), *(rng.randrange(1, (1 << 28) // w) * w - 1 for _ in range(2000))]:
            assert lib.quotient(n, w) == n // w
