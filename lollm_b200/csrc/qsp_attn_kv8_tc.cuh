// Shared by the tensor-core kernels of the 8-bit cache: bounded waits, operand descriptors and MMAs on
// 8-bit floats, TMEM reads, and the warps that load tiles and scales. Each including file has its own error flag.
#pragma once

#include <limits.h>

#include "qsp_attn_kv8.cuh"
#include "qsp_tc.cuh"

namespace qsp {
namespace kv8 {

static __device__ int g_kv8_error = 0;

constexpr int CODE_WAIT = 302;       // a bounded wait ran out
constexpr float SLACK = 4.f;         // log2 units the running maximum may lag behind
constexpr float BIAS = 11.f;         // weights are held times 2^BIAS: at most 2^(SLACK + BIAS) = 32768, under e5m2's 57344
constexpr float NOTHING = -1e30f;    // maximum of a row that has seen nothing

// A piece of work as the scales' warp hands it to the others, which run up to 4 tiles behind it (and the
// slowest of them 3 pieces more): 8 slots.
constexpr int NDESC = 8;
struct Desc {
  int b, row0, g, j0;         // sequence, first row of the unit, kv head, first tile
  int n, base, slot, whole;   // tiles (0: no more pieces), sequence length, partial's slot, whole unit
};

// ---------------------------------------------------------------- descriptors
// rows of W bytes (16, 32, 64 or 128), swizzled over W bytes, 8-row groups 8·W apart: the layout of
// TMA boxes with inner extent W. K-major: rows are M/N, bytes along the row K. MN-major: the row is
// M/N, rows are K; lead = distance of the next W elements along M/N (0: the same again).
struct Sdesc {   // the address is in the low word; all offsets within shared memory are added there
  uint32_t lo, hi;
};
template <int W>
__device__ __forceinline__ Sdesc sdesc(const void* p, uint32_t lead) {
  constexpr uint32_t type = W == 128 ? 2 : W == 64 ? 4 : W == 32 ? 6 : 0;
  return {((tc::smem_u32(p) & 0x3FFFFu) >> 4) | (lead >> 4) << 16, (8 * W >> 4) | 1u << 14 | type << 29};
}
template <int W>
__device__ __forceinline__ int swz(int row, int chunk) {   // byte offset of a 16-byte chunk of a row
  constexpr int M = W / 16 - 1;
  return row * W + ((chunk ^ (row * W / 128 & M)) << 4);
}
// kind::f8f6f4, D fp32, A e4m3, B e4m3 or e5m2
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N, bool mn_major, bool b_e5m2) {
  return (1u << 4) | (b_e5m2 ? 1u << 10 : 0u) | (mn_major ? 3u << 15 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// `STEPS` MMAs of K = 32 into the same accumulator, the operands' addresses a_step and b_step (in
// 16-byte units) apart; the first accumulates iff acc != 0. Issued by a converged warp.
template <int STEPS, int A_STEP, int B_STEP>
__device__ __forceinline__ void umma_f8_warp(uint32_t d, Sdesc a, Sdesc b, uint32_t idesc, uint32_t acc) {
  static_assert(STEPS == 1 || STEPS == 2 || STEPS == 4, "");
  if constexpr (STEPS == 4) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t"
        "setp.eq.b32 p, %6, %6;\n\t"
        "add.u32 x, %1, %7;\n\tadd.u32 y, %3, %8;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t"
        "add.u32 x, x, %7;\n\tadd.u32 y, y, %8;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t"
        "add.u32 x, x, %7;\n\tadd.u32 y, y, %8;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t}" ::"r"(d),
        "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(acc), "n"(A_STEP), "n"(B_STEP)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 a, b;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t}" ::"r"(d),
        "r"(a.lo), "r"(a.hi), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(acc)
        : "memory");
    if constexpr (STEPS == 2)
      umma_f8_warp<1, A_STEP, B_STEP>(d, {a.lo + A_STEP, a.hi}, {b.lo + B_STEP, b.hi}, idesc, 1);
  }
}

// ---------------------------------------------------------------- waits
// Bounded; the poll is kept small (five roles share an instruction cache), the rest is out of line.
static __device__ __noinline__ bool give_up(uint32_t polls, volatile int* abort) {
  if (*abort) return true;
  if (polls < tc::WAIT_LIMIT) {
    __nanosleep(64);
    return false;
  }
  atomicExch(&g_kv8_error, CODE_WAIT);
  *abort = 1;
  return true;
}
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
  uint32_t n = 0;
#pragma unroll 1
  while (!tc::mbar_try_wait(bar, parity))
    if ((++n & 255u) == 0 && give_up(n, abort)) return;
}

// ---------------------------------------------------------------- TMEM, 8 columns of this warp's 32 lanes
__device__ __forceinline__ void tm_ld8(uint32_t t, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(t));
}
__device__ __forceinline__ void tm_st8(uint32_t t, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// the registers are operands, so that nothing reads them before the wait
__device__ __forceinline__ void tm_wait_ld8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void tm_wait_ld8(uint32_t (&r)[8], uint32_t (&s)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(s[0]), "+r"(s[1]),
                 "+r"(s[2]), "+r"(s[3]), "+r"(s[4]), "+r"(s[5]), "+r"(s[6]), "+r"(s[7])::"memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + 2^(-x·log2(e))): off by 2^-17 relative at x = -80 (the rounded product), 2^-21 near 0. A bf16 output
// needs no more, and the exact quotient's code is ten times as long.
__device__ __forceinline__ float sigmoid_ex2(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + ex2(x * -LOG2E)));
  return y;
}
__device__ __forceinline__ uint16_t half2_to_e4m3x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return r;
}
// ---------------------------------------------------------------- softmax weights as sums of e5m2 values
// A weight w >= 0, rounded to fp16, is cut into three e5m2 values: the upper byte of an fp16 value is the e5m2 value below it,
// so a = upper byte(w), b = upper byte(S·(w − a)), c = S·(w − a) − b rounded to one, and w = a + (b + c) / S. Every part keeps
// 3 bits or more of what is left, so w is off by at most 2^-9 of its power of two (half a bf16 step is 2^-8), or by
// 2^-17 / S where that is more: 2^-28 / S of a row's largest, which is held as 2^BIAS at least. The relative precision of
// bf16 thus reaches down to 2^-20 / S of the largest. (Two e4m3 values reached 2^-10, and were 0 under 2^-18: one key with
// most of the weight and 32k weak ones lost what the weak ones add up to, 6 to 60 per cent of the output.)
// The subtractions are exact; no conversion is needed, which an SM does at a quarter of the rate or less.
template <int S>
__device__ __forceinline__ void split_weights(__half2 w, uint32_t& a, uint32_t& b, uint32_t& c) {   // pairs; parts are upper bytes
  auto upper = [](uint32_t x) {
    x &= 0xff00ff00u;
    return *reinterpret_cast<__half2*>(&x);
  };
  auto bits = [](__half2 x) { return *reinterpret_cast<uint32_t*>(&x); };
  a = bits(w);
  __half2 r = __hsub2(w, upper(a));
  if constexpr (S != 1) r = __hmul2(r, __float2half2_rn((float)S));
  b = bits(r);
  c = bits(__hsub2(r, upper(b))) + 0x00800080u;   // half of the upper byte's last place: no carry out of a value
}
__device__ __forceinline__ uint32_t upper_bytes(uint32_t x, uint32_t y) { return __byte_perm(x, y, 0x7531); }   // of two pairs

__device__ __forceinline__ void bar_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool bar_any(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)p)
      : "memory");
  return r != 0;
}

constexpr uint32_t MISSING = 0xffffu;   // scale exponents of a key that has no page

// ---------------------------------------------------------------- the loading warps
// a box at (x, row) under an L2 policy; issued by a converged warp
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int row, uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;\n\t}" ::"r"(
          tc::smem_u32(dst)),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(row), "l"(policy)
      : "memory");
}
// K or V tiles of the CTA's pieces into a ring of `slots`, by TMA: boxes of box_rows keys x CW bytes; lane i looks
// up the page of the tile's i-th box_rows keys, one tile ahead. once: see read_once.
// Is a tile read by one CTA only? Not where a unit's keys are another row group's too, nor where the pool has fewer pages
// than the table has entries, so that sequences share some (a common prefix). Evict-first keeps what is read once from
// driving queries, page tables and partials out of L2 (64 x 4 tokens over 2k keys 34.7 us, 37.8 without; over 1k to 32k 174 and
// 182), but drives shared pages out too (64 x 4 over the same 32k keys 264 us, 248 without; the same 120k 1234 and 1083).
__device__ __forceinline__ bool read_once(const qsp_attn_kv8_layer& L, int n_rg) {
  return n_rg == 1 && L.num_pages >= (int64_t)L.batch * L.max_pages;
}
template <int HD, int CW, typename PieceAt>
__device__ __forceinline__ void load_tiles(const qsp_attn_kv8_layer& L, const CUtensorMap* map, uint8_t* ring, uint64_t* full,
                                           uint64_t* empty, int slots, int box_rows, bool once, const PieceAt& piece_at,
                                           volatile int* abort) {
  const int lane = threadIdx.x & 31, cap = L.max_pages * L.page_size;
  const int chunks = TILE / box_rows, pages_step = TILE / L.page_size, slot_step = TILE % L.page_size;
  int slot = 0;
  uint32_t turn = 1;   // parity of "empty" for this turn of the ring
  uint64_t policy;     // what is read once stays out of the way of queries, page tables and partials in L2
  if (once) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  for (uint32_t piece = 0;; ++piece) {
    const Desc p = piece_at(piece);
    if (p.n == 0) break;
    const int kv_end = min(p.base + L.tokens, cap);
    const int32_t* pages = L.page_table + (int64_t)p.b * L.max_pages;
    int key = lane < chunks ? p.j0 * TILE + lane * box_rows : INT_MAX - 2 * TILE;   // this lane's first key of the tile
    int lp = key / L.page_size, in = key - lp * L.page_size;
    int page = key < kv_end ? pages[lp] : -1;
    for (int j = 0; j < p.n; ++j) {
      // row of the pages' [pages·n_kv·page_size, hd] view, or -1
      const int row = page >= 0 && page < L.num_pages ? (page * L.n_kv_heads + p.g) * L.page_size + in : -1;
      if (lane < chunks) key += TILE;
      lp += pages_step;
      in += slot_step;
      if (in >= L.page_size) {
        in -= L.page_size;
        ++lp;
      }
      page = j + 1 < p.n && key < kv_end ? pages[lp] : -1;
      wait_bar(&empty[slot], turn, abort);
      __syncwarp();
      const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
      tc::mbar_expect_tx_warp(&full[slot], __popc(there) * box_rows * HD);
      uint8_t* dst = ring + slot * (TILE * HD);
      for (int i = 0; i < chunks; ++i, dst += box_rows * CW) {
        const int r = __shfl_sync(0xffffffffu, row, i);
        if (r >= 0) {
#pragma unroll
          for (int cb = 0; cb < HD / CW; ++cb) load_box(dst + cb * (TILE * CW), map, &full[slot], cb * CW, r, policy);
        }
      }
      if (++slot == slots) {
        slot = 0;
        turn ^= 1u;
      }
    }
  }
}

// ---------------------------------------------------------------- the scales' warp
// Walks through the CTA's share of the work and describes its pieces to the other warps; brings the scales of
// each tile's keys (lane i: keys i, 32 + i, 64 + i, 96 + i), in step with the K ring of `slots`, and hands them to
// put(). Pages are loaded two tiles ahead, scales one. A tile's scales go into a ring two longer than K's: when
// they are written, QK of the tile `slots` before is done, so it had been issued, after the scores of the
// tile before that, or of its predecessor, had been read. Returns the last piece.
struct Scales {
  float ks[4], vs[4];
  bool here[4];   // the key has a page
};
template <typename Put>
__device__ __forceinline__ Piece walk_and_scales(const qsp_attn_kv8_layer& L, int n_rg, int rows, int slots, Walk& w, Desc* desc,
                                                 uint64_t* dfull, uint64_t* kfull, uint64_t* kempty, volatile int* abort,
                                                 const Put& put) {
  const int lane = threadIdx.x & 31, cap = L.max_pages * L.page_size;
  const int nb = L.page_size / L.scale_block, sb_log = __ffs(L.scale_block) - 1;
  const int pages_step = TILE / L.page_size, slot_step = TILE % L.page_size;
  int slot = 0;
  uint32_t turn = 1;
  Piece p;
  p.n = 0;
  for (uint32_t piece = 0;; ++piece) {
    const bool more = next_piece<TILE>(L, n_rg, rows, w, p);
    const int base = more ? min(p.len, cap) : 0;
    if (lane == 0) {
      desc[piece % NDESC] = {p.b, p.rg * rows, p.g, p.j0, more ? p.n : 0, base, p.slot(), p.whole()};
      tc::mbar_arrive(&dfull[piece % NDESC]);
    }
    if (!more) break;
    const int kv_end = min(base + L.tokens, cap);
    const int32_t* pages = L.page_table + (int64_t)p.b * L.max_pages;
    int page[4], blk[4], lp[4], in[4];   // of tile j + 1, then j + 2
    Scales x;                            // of tile j
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = p.j0 * TILE + i * 32 + lane;
      lp[i] = key / L.page_size;
      in[i] = key - lp[i] * L.page_size;
    }
    auto pages_at = [&](int j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        blk[i] = in[i] >> sb_log;
        page[i] = j < p.n && (p.j0 + j) * TILE + i * 32 + lane < kv_end ? pages[lp[i]] : -1;
        lp[i] += pages_step;
        in[i] += slot_step;
        if (in[i] >= L.page_size) {
          in[i] -= L.page_size;
          ++lp[i];
        }
      }
    };
    auto scales_at = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.here[i] = page[i] >= 0 && page[i] < L.num_pages;
        const int64_t at = x.here[i] ? ((int64_t)page[i] * L.n_kv_heads + p.g) * nb + blk[i] : 0;
        x.ks[i] = L.k_scales[at];
        x.vs[i] = L.v_scales[at];
      }
    };
    pages_at(0);
    scales_at();
    pages_at(1);
    for (int j = 0; j < p.n; ++j) {
      wait_bar(&kempty[slot], turn, abort);
      put(x);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&kfull[slot]);
      if (++slot == slots) {
        slot = 0;
        turn ^= 1u;
      }
      scales_at();
      pages_at(j + 2);
    }
  }
  return p;
}

}  // namespace kv8
}  // namespace qsp
