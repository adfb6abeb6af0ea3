// Attention over the 8-bit KV cache for many query rows (chunks of prompts) on tcgen05 tensor cores: bf16
// models, page sizes and scale blocks that are a multiple of 8, more than 64 rows (tokens x heads of the kv head).
//
// A unit is 128 query rows, which are the rows of the products:
//   S [128, 128 keys] = Q [128, hd] · K^T       A = Q from shared memory, B = K as it lies in the cache
//   O [128, hd]      += P [128, 128 keys] · V   A = P from TMEM,          B = V read along its rows
// The codes of K and V are operands as they are. Q (times a power of two per row) is the sum of an e4m3 and an
// e5m2 value, hi = e4m3(q), lo = e5m2(q - hi), which accumulate into the same S: hi holds the upper 4 bits; what is
// left is at most 8 units of a bf16's last place, which e5m2's 3 bits hold exactly, for elements down to 2^-6, of a
// row whose largest is scaled to 224..448; smaller ones are off by at most 2^-14, 2^-21 of the largest. A softmax weight
// is the sum of three e5m2 values (split_weights, unscaled: they accumulate into the same O), which is bf16's
// precision down to 2^-20 of the row's largest.
//
// A row of S is one lane of TMEM: two threads have 64 of its keys each, warps i and 4 + i the same 32 rows.
// They need not know the maximum exactly: m is raised, and O rescaled, only when a score passes it by more
// than 2^SLACK, which the two warps learn from one barrier with a vote. The scales of the keys multiply
// the scores, those of the values are added to them as log2 units (so that O's weights are p·vscale, at
// most 2^SLACK, and the sum takes them back). 8 keys share their scales, so an exponent is one fused multiply-add of
// a score. (Scales of single keys: 1500 of a tile's cycles were their reads from shared memory.)
//
// QK of a tile runs while the weights of the one before are computed (its scores are in registers by then),
// and the weights' product after it.
//
// A tile takes 1024 + 1350 cycles of the tensor cores at hd 256 (two parts of Q, three of P) and 2100 of the softmax: 64
// exponentials a thread at 16 an SM and cycle are half of that. They overlap but for the start of each; about 3300
// cycles were measured, and 2700 with weights of two parts, whose small ones were lost (8 sequences x 127 tokens over 1k
// to 2k keys, 2 kv heads of 256, 48 and 53 us; 2 x 512 over 8k 119 and 141 to 154 us). At head sizes up to 128, where
// TMEM has room for the weights of two tiles, the third part costs nothing (8 x 127 of size 64: 28 us). Against 64
// rows a unit (tc_kernel in groups): 8 x 127 72 -> 52 us, 64 x 16 over 2k 87 -> 58, 4 x 2048 from an empty cache 451 -> 315,
// 27 x 64 tokens of 4 and 2 heads over 4k to 9k 88 -> 77.
#include "qsp_attn_kv8_tc.cuh"

#include <algorithm>

namespace qsp {
namespace kv8 {

constexpr int RR = 128;    // rows of a unit

template <int HD>
struct RowsCfg {
  static constexpr int CW = HD < 128 ? HD : 128, CB = HD / CW;   // bytes of a swizzled row, column blocks
  static constexpr int SLOT = TILE * HD, QB = 2 * RR * HD;       // a K or V tile; hi and lo of Q
  // barriers, piece descriptors, share()'s ints, row scales (of two pieces), maxima and sums of the halves, flag
  static constexpr int SMALL = 8 * 34 + NDESC * 32 + 4 * 68 + 4 * (2 * RR + 4 * RR) + 16;
  static constexpr int SCALES = TILE / GROUP * 16 + 16;          // of a tile: {K, log2 of V, 1 / V} of 8 keys; are keys missing
  static constexpr int CH = HD < 64 ? HD / 2 : 32;               // columns of O that a warp brings out at a time, 16 rows
  static constexpr int OUT = 8 * 16 * (CH + 4) * 4;
  static constexpr size_t bytes(int ns) { return (size_t)ns * SLOT + QB + OUT + SMALL + (ns / 2 + 2) * SCALES; }
  static constexpr int slots() {
    int ns = 8;
    while (bytes(ns) > 232448) --ns;
    return ns;
  }
  static constexpr int NS = slots(), NSK = NS / 2, NSV = NS - NSK, NSE = NSK + 2;
  static constexpr size_t BYTES = bytes(NS);
  static constexpr int SOFTMAX = 256, THREADS = SOFTMAX + 128;
  // TMEM columns: scores, weights (of two tiles where O leaves room), output
  static constexpr int NP = HD <= 128 ? 2 : 1, PW = 96, S = 0, P = 128, O = 512 - (HD <= 128 ? 128 : HD), COLS = 512;
  static_assert(P + NP * PW <= O, "the weights run into O");
  static_assert(NSK >= 2 && NSK <= 4, "ring too short, or too long for the descriptors' slots");
};

// kind::f8f6f4, D fp32, A e4m3 or e5m2, B e4m3
__host__ __device__ constexpr uint32_t idesc_rows(int N, bool a_e5m2, bool b_mn_major) {
  return (1u << 4) | (a_e5m2 ? 1u << 7 : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// K = 32 keys: D [128, N] += A (TMEM, 8 columns) · B. Issued by a converged warp.
__device__ __forceinline__ void umma_ts_warp(uint32_t d, uint32_t a, Sdesc b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t.reg .b64 b;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b.lo), "r"(b.hi), "r"(idesc), "r"(acc)
      : "memory");
}

#define QSP_O16(x, o)                                                                                                       \
  "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7]), \
      "=r"(x[o + 8]), "=r"(x[o + 9]), "=r"(x[o + 10]), "=r"(x[o + 11]), "=r"(x[o + 12]), "=r"(x[o + 13]), "=r"(x[o + 14]),  \
      "=r"(x[o + 15])
#define QSP_I16(x, o)                                                                                                       \
  "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7]),          \
      "r"(x[o + 8]), "r"(x[o + 9]), "r"(x[o + 10]), "r"(x[o + 11]), "r"(x[o + 12]), "r"(x[o + 13]), "r"(x[o + 14]), "r"(x[o + 15])
// 64 or 16 columns of this warp's 32 lanes, there when the statement ends
__device__ __forceinline__ void tm_ld64(uint32_t t, uint32_t (&x)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,"
      "%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : QSP_O16(x, 0), QSP_O16(x, 16), QSP_O16(x, 32), QSP_O16(x, 48)
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t t, uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : QSP_O16(x, 0)
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t t, const uint32_t (&x)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
               QSP_I16(x, 0)
               : "memory");
}
#undef QSP_O16
#undef QSP_I16

// pairs of fp32: one instruction for both
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ uint16_t half2_to_e5m2x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return r;
}
// the two warps that share rows
__device__ __forceinline__ void pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)p)
      : "memory");
  return r != 0;
}

template <int HD>
__global__ void __launch_bounds__(RowsCfg<HD>::THREADS, 1)
rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const qsp_attn_kv8_layer L, int n_rg,
            int box_rows, bool vec) {
  using C = RowsCfg<HD>;
  constexpr int NSK = C::NSK, NSV = C::NSV, NSE = C::NSE, CW = C::CW, CB = C::CB, EPL = HD / 32;
  extern __shared__ __align__(1024) uint8_t sK[];                // the swizzles go by address: 1024-byte tiles
  uint8_t* sV = sK + NSK * C::SLOT;
  uint8_t* sQ = sV + NSV * C::SLOT;                              // [hi | lo][column block][128 rows][CW]
  float* stage = reinterpret_cast<float*>(sQ + C::QB);           // [8 warps][16 rows][CH + 4] of O
  float4* sc = reinterpret_cast<float4*>(sQ + C::QB + C::OUT);   // [NSE][16] K scale, log2 of V scale + BIAS, 1 / V scale
  int* holes = reinterpret_cast<int*>(sc + NSE * (TILE / GROUP));   // [NSE] (16 bytes each): keys are missing
  uint64_t* kfull = reinterpret_cast<uint64_t*>(holes + NSE * 4);
  uint64_t* kempty = kfull + NSK;
  uint64_t* vfull = kempty + NSK;
  uint64_t* vempty = vfull + NSV;
  uint64_t* sfull = vempty + NSV;  // scores of a tile are in TMEM
  uint64_t* sread = sfull + 1;     // ... and in registers
  uint64_t* pfull = sread + 1;     // weights of a tile are in TMEM
  uint64_t* pdone = pfull + 2;     // ... and their product with V is done
  uint64_t* qfull = pdone + 2;     // Q of a piece is in shared memory
  uint64_t* dfull = qfull + 1;     // [NDESC] a piece's descriptor is there; 2·8 + 7 + 8 barriers at most
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kfull + 33);
  Desc* desc = reinterpret_cast<Desc*>(kfull + 34);
  int* sh = reinterpret_cast<int*>(desc + NDESC);                // [68] for share()
  float* qs = reinterpret_cast<float*>(sh + 68);                 // [2][128] scale of a row's scores, in log2 units, by piece
  float* half_max = qs + 2 * RR;                                 // [2][128]
  float* half_sum = half_max + 2 * RR;                           // [2][128]
  volatile int* abort = reinterpret_cast<volatile int*>(half_sum + 2 * RR);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int W_K = 8, W_V = 9, W_E = 10, W_MMA = 11;
  const int nrep = L.n_heads / L.n_kv_heads, rows_total = nrep * L.tokens;

  if (tid == 0) {
    for (int i = 0; i < 2 * C::NS; ++i) tc::mbar_init(&kfull[i], i < NSK ? 2 : 1);   // kfull (K and its scales), kempty, vfull, vempty
    tc::mbar_init(sfull, 1);
    tc::mbar_init(sread, 8);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&pfull[i], 8);
      tc::mbar_init(&pdone[i], 1);
    }
    tc::mbar_init(qfull, 8);
    for (int i = 0; i < NDESC; ++i) tc::mbar_init(&dfull[i], 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (lane == 0 && (warp == W_K || warp == W_V))
    asm volatile("prefetch.tensormap [%0];" ::"l"(warp == W_K ? &tmK : &tmV) : "memory");
  pdl_wait();
  // TMEM between the previous kernel's end and the next one's start: as in tc_kernel
  if (warp == W_MMA) {
    tc::tmem_alloc(tmem_slot, C::COLS);
    tc::fence_before();
  }
  Walk w = share<TILE>(L, n_rg, RR, sh);
  pdl_trigger();
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  auto piece_at = [&](uint32_t i) -> Desc {   // the i-th piece of this CTA
    wait_bar(&dfull[i % NDESC], i / NDESC & 1u, abort);
    __syncwarp();
    Desc d = desc[i % NDESC];
    if (__any_sync(0xffffffffu, *abort)) d.n = 0;   // a wait ran out: what is there may not be a descriptor
    return d;
  };

  if (warp == W_K || warp == W_V) {
    const bool is_v = warp == W_V;
    load_tiles<HD, CW>(L, is_v ? &tmV : &tmK, is_v ? sV : sK, is_v ? vfull : kfull, is_v ? vempty : kempty, is_v ? NSV : NSK, box_rows,
                       read_once(L, n_rg), piece_at, abort);
  } else if (warp == W_E) {
    int slot = 0;
    const Piece p = walk_and_scales(L, n_rg, RR, NSK, w, desc, dfull, kfull, kempty, abort, [&](const Scales& x) {
      bool all = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // a group has a page if its first key has
        all = all && x.here[i];
        if (lane % GROUP == 0)
          sc[slot * (TILE / GROUP) + (i * 32 + lane) / GROUP] =
              x.here[i] ? make_float4(x.ks[i], (float)exp_of(x.vs[i]) + BIAS, exp2i(-exp_of(x.vs[i])), 0.f) : make_float4(0.f, -INFINITY, 0.f, 0.f);
      }
      all = __all_sync(0xffffffffu, all);
      if (lane == 0) holes[slot * 4] = !all;
      if (++slot == NSE) slot = 0;
    });
    if (lane == 0) put_meta(scratch(L, gridDim.x, RR), w, p);
  } else if (warp == W_MMA) {
    // ---------------- products, in the order QK(0) QK(1) PV(0) QK(2) PV(1) ... of each piece. QK(t) overwrites the
    // scores of t - 1 once they are in registers. With two buffers the weights of t go where those of t - 2 were:
    // their product was issued before QK(t), whose scores the softmax has waited for. With one the softmax waits for
    // the product of t - 1, which is done long before.
    constexpr int STEP = 32 * CW / 16;   // 32 keys of V
    constexpr uint32_t QK_HI = idesc_rows(TILE, false, false), QK_LO = idesc_rows(TILE, true, false);
    constexpr uint32_t ID_PV = idesc_rows(CW, true, true);
    const Sdesc dK = sdesc<CW>(sK, 16), dV = sdesc<CW>(sV, 0), dQ = sdesc<CW>(sQ, 16);
    uint32_t tile = 0, kslot = 0, kturn = 0, vslot = 0, vturn = 0;
    for (uint32_t piece = 0;; ++piece) {
      const int n = piece_at(piece).n;
      if (n == 0) break;
      wait_bar(qfull, piece & 1u, abort);
      auto qk = [&](uint32_t t) {
        if (t > 0) wait_bar(sread, (t - 1) & 1u, abort);
        wait_bar(&kfull[kslot], kturn, abort);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int cb = 0; cb < CB; ++cb)
            umma_f8_warp<CW / 32, 2, 2>(tmem + C::S, {dQ.lo + (part * RR * HD + cb * RR * CW) / 16, dQ.hi},
                                          {dK.lo + (kslot * C::SLOT + cb * (TILE * CW)) / 16, dK.hi}, part ? QK_LO : QK_HI, part + cb > 0);
        tc::umma_commit_warp(&kempty[kslot]);
        tc::umma_commit_warp(sfull);
        if (++kslot == NSK) {
          kslot = 0;
          kturn ^= 1u;
        }
      };
      qk(tile);
      for (int j = 0; j < n; ++j, ++tile) {
        if (j + 1 < n) qk(tile + 1);
        const uint32_t pb = tile & 1;
        wait_bar(&vfull[vslot], vturn, abort);
        wait_bar(&pfull[pb], (tile >> 1) & 1u, abort);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int mb = 0; mb < CB; ++mb)
#pragma unroll
          for (int s = 0; s < 12; ++s) {   // 4 steps of 32 keys, three parts
            const int k = s / 3, part = s % 3;
            umma_ts_warp(tmem + C::O + mb * CW, tmem + C::P + pb % C::NP * C::PW + (k >> 1) * 48 + part * 16 + (k & 1) * 8,
                         {dV.lo + (vslot * C::SLOT + mb * (TILE * CW)) / 16 + k * STEP, dV.hi}, ID_PV, j > 0 || s > 0);
          }
        tc::umma_commit_warp(&vempty[vslot]);
        tc::umma_commit_warp(&pdone[pb]);
        if (++vslot == NSV) {
          vslot = 0;
          vturn ^= 1u;
        }
      }
    }
  } else {
    // ---------------- softmax: thread = row of the unit, 64 of a tile's keys
    const int half = warp >> 2, wq = warp & 3, row = wq * 32 + lane, bar = 1 + wq;
    const uint32_t tlane = tmem + ((uint32_t)(wq * 32) << 16);
    const Scratch ws = scratch(L, gridDim.x, RR);
    uint32_t tile = 0, piece = 0, eslot = 0, vslot = 0, vturn = 0;

    // Q of a piece: a warp per row, four rows while the next eight are loaded. (A loop: as straight code it took three
    // times as long, for the fetching of instructions.)
    auto stage_q = [&](const Desc& q, uint32_t n) {
      int64_t at = -1;   // of row lane·8 + warp in q_buf
      if (lane < 16 && q.row0 + lane * 8 + warp < rows_total) {
        const int rr = q.row0 + lane * 8 + warp, t = rr / nrep;
        at = (((int64_t)q.b * L.tokens + t) * L.n_heads + q.g * nrep + rr - t * nrep) * HD;
      }
      Row<__nv_bfloat16, EPL> x[4], y[4], z[4];
      auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t from = __shfl_sync(0xffffffffu, at, i0 + i);
          z[i].zero();
          if (from >= 0) z[i].load(static_cast<const __nv_bfloat16*>(L.q_buf) + from, lane, true);
        }
      };
      const int byte = lane * EPL, in = byte % CW;
      load(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = z[i];
      load(4);
#pragma unroll 1
      for (int i0 = 0; i0 < 16; i0 += 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i], y[i] = z[i];
        if (i0 < 8) load(i0 + 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (i0 + i) * 8 + warp;
          const uint32_t top = __reduce_max_sync(0xffffffffu, x[i].top());
          const bool fine = top < NOT_FINITE;
          const int e = fine ? scale_exp(top) : 0;
          const float inv = exp2i(-e);
          uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
          for (int k = 0; k < EPL; k += 2) {
            const __half2 v = __floats2half2_rn(x[i][k] * inv, EPL > 1 ? x[i][EPL > 1 ? k + 1 : 0] * inv : 0.f);
            const uint16_t h = half2_to_e4m3x2(v);
            hi[k / 4] |= (uint32_t)h << (k % 4 * 8);
            lo[k / 4] |= (uint32_t)half2_to_e5m2x2(__hsub2(v, e4m3x2_to_half2(h))) << (k % 4 * 8);
          }
          if (!fine) hi[0] = hi[1] = lo[0] = lo[1] = 0;   // the scale says NaN
          uint8_t* dst = sQ + byte / CW * (RR * CW) + swz<CW>(r, in / 16) + in % 16;
          store_bytes<EPL>(dst, hi[0], hi[1]);
          store_bytes<EPL>(dst + RR * HD, lo[0], lo[1]);
          if (lane == 0) qs[(n & 1) * RR + r] = fine ? exp2i(e) * (L.scale * LOG2E) : NAN;
        }
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(qfull);
    };
    // the two warps of a pair meet at its barrier, so they have to agree on the next piece (they do, but for
    // a wait that ran out in one of them)
    auto agreed_piece_at = [&](uint32_t i) -> Desc {
      Desc d = piece_at(i);
      if (pair_any(bar, d.n == 0)) d.n = 0;
      return d;
    };
    auto prefetch_row = [&](const __nv_bfloat16* base, const Desc& q, int64_t ld, int stride, int off) {   // half of this thread's row
      const int r = q.row0 + row, tt = r / nrep;
      if (r < rows_total) {
        const __nv_bfloat16* at = base + ((int64_t)q.b * L.tokens + tt) * ld + (int64_t)(q.g * nrep + r - tt * nrep) * stride + off + half * (HD / 2);
#pragma unroll
        for (int i = 0; i < HD / 2; i += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i));
      }
    };
    Desc p;
    float m, l;
    for (;; ++piece) {
      // The scores of the last tile are here, so Q is free for the next piece, whose first product then runs beside the
      // rest of this one: O out of TMEM, half of the columns each.
      const Desc next = agreed_piece_at(piece);
      if (next.n > 0) stage_q(next, piece);
      if (piece > 0) {
        half_sum[half * RR + row] = l;
        pair_sync(bar);
        const float sum = half_sum[row] + half_sum[RR + row], inv = p.whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
        if (!p.whole && half == 0) ws.ml[(int64_t)p.slot * RR + row] = make_float2(sum == 0.f ? -INFINITY : m, sum);
        // 16 rows x CH columns at a time through shared memory, so that a warp's accesses to gate and output are runs
        // of CH elements: lane = 8 columns of row (pass, lane / LPR)
        constexpr int CH = C::CH, LPR = CH / 8, PASSES = LPR / 2, ROWS = 2 * PASSES;
        float* st = stage + warp * (16 * (CH + 4));
        const int c0 = half * (HD / 2), my_col = c0 + lane % LPR * 8;
        const __nv_bfloat16* gate[ROWS];
        __nv_bfloat16* out[ROWS];
        bool real[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int mine = p.row0 + wq * 32 + i / PASSES * 16 + i % PASSES * (32 / LPR) + lane / LPR, tt = mine / nrep, hq = p.g * nrep + mine - tt * nrep;
          const int64_t mrow = (int64_t)p.b * L.tokens + tt;
          real[i] = mine < rows_total;
          gate[i] = static_cast<const __nv_bfloat16*>(L.qkv) + mrow * L.ld_qkv + (int64_t)hq * 2 * HD + HD + my_col;
          out[i] = static_cast<__nv_bfloat16*>(L.out) + mrow * L.ld_out + (int64_t)hq * HD + my_col;
        }
        Row<__nv_bfloat16, 8> g[ROWS];
        auto load_gates = [&](int c) {
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            g[i].zero();
            if (p.whole && real[i]) g[i].load(gate[i] + c, 0, vec);
          }
        };
        load_gates(0);
        wait_bar(&pdone[(tile - 1) & 1], ((tile - 1) >> 1) & 1, abort);
        __syncwarp();
        tc::fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 2; c += CH) {
          float o[CH];
#pragma unroll
          for (int k = 0; k < CH; k += 16) {
            uint32_t u[16];
            tm_ld16(tlane + C::O + c0 + c + k, u);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[k + i] = __uint_as_float(u[i]) * inv;
          }
          Row<__nv_bfloat16, 8> now[ROWS];
#pragma unroll
          for (int i = 0; i < ROWS; ++i) now[i] = g[i];
          if (c + CH < HD / 2) load_gates(c + CH);
#pragma unroll
          for (int i = 0; i < ROWS; ++i) {
            if (i % PASSES == 0) {
              __syncwarp();
              if (lane / 16 == i / PASSES) {
#pragma unroll
                for (int k = 0; k < CH; k += 4) *reinterpret_cast<float4*>(st + lane % 16 * (CH + 4) + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
              }
              __syncwarp();
            }
            const int r = i % PASSES * (32 / LPR) + lane / LPR;
            const float4 a = *reinterpret_cast<const float4*>(st + r * (CH + 4) + lane % LPR * 8), b = *reinterpret_cast<const float4*>(st + r * (CH + 4) + lane % LPR * 8 + 4);
            if (!p.whole) {
              float* to = ws.o + ((int64_t)p.slot * RR + wq * 32 + i / PASSES * 16 + r) * HD + my_col + c;
              *reinterpret_cast<float4*>(to) = a;
              *reinterpret_cast<float4*>(to + 4) = b;
            } else if (real[i]) {
              const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
              __nv_bfloat162 y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) y[k] = __floats2bfloat162_rn(v[2 * k] * sigmoid_ex2(now[i][2 * k]), v[2 * k + 1] * sigmoid_ex2(now[i][2 * k + 1]));
              if (vec) {
                const uint32_t* u = reinterpret_cast<const uint32_t*>(y);
                *reinterpret_cast<uint4*>(out[i] + c) = make_uint4(u[0], u[1], u[2], u[3]);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) out[i][c + 2 * k] = __low2bfloat16(y[k]), out[i][c + 2 * k + 1] = __high2bfloat16(y[k]);
              }
            }
            __syncwarp();
          }
        }
        tc::fence_before();   // the next piece's products overwrite O after its pfull
      }
      if (next.n == 0) break;
      p = next;
      const int rr = p.row0 + row, t = rr / nrep;
      const int kv_end = min(p.base + L.tokens, L.max_pages * L.page_size);
      int sees = p.base + t - p.j0 * TILE - half * 64;   // the last key of this thread's 64 that the row sees
      float q_scale = 0.f;
      m = NOTHING;
      l = 0.f;
      for (int j = 0; j < p.n; ++j, ++tile, sees -= TILE) {
        if (j == p.n - 1) {
          // into L2: the gates of this piece, Q of the next
          if (p.whole) prefetch_row(static_cast<const __nv_bfloat16*>(L.qkv), p, L.ld_qkv, 2 * HD, HD);
          const Desc q = piece_at(piece + 1);
          if (q.n > 0) prefetch_row(static_cast<const __nv_bfloat16*>(L.q_buf), q, (int64_t)L.n_heads * HD, HD, 0);
        }
        wait_bar(sfull, tile & 1u, abort);
        __syncwarp();
        tc::fence_after();
        if (j == 0) q_scale = qs[(piece & 1) * RR + row];   // (staged before QK, by another warp)
        float d[64];
        {
          uint32_t x[64];
          tm_ld64(tlane + C::S + half * 64, x);
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(sread);
#pragma unroll
          for (int k = 0; k < 64; ++k) d[k] = __uint_as_float(x[k]);
        }
        const float4* s = sc + eslot * (TILE / GROUP) + half * (64 / GROUP);
        const bool gaps = holes[eslot * 4] != 0;
        if (++eslot == NSE) eslot = 0;
        // exponents of the weights, relative to the maximum so far
        const float ref = m == NOTHING ? 0.f : m;
#pragma unroll
        for (int g = 0; g < 64 / GROUP; ++g) {
          const float4 c = s[g];
          const float2 scale = make_float2(c.x * q_scale, c.x * q_scale), off = make_float2(c.y - ref, c.y - ref);
#pragma unroll
          for (int k = g * GROUP; k < (g + 1) * GROUP; k += 2) {
            const float2 y = fma2(make_float2(d[k], d[k + 1]), scale, off);
            d[k] = y.x, d[k + 1] = y.y;
          }
        }
        if (gaps || __any_sync(0xffffffffu, sees < 63)) {
#pragma unroll
          for (int g = 0; g < 64 / GROUP; ++g) {
            const bool there = s[g].y != -INFINITY;
#pragma unroll
            for (int k = g * GROUP; k < (g + 1) * GROUP; ++k)
              if (k > sees || !there) d[k] = -INFINITY;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 64; k += 2) top = fmaxf(top, fmaxf(d[k], d[k + 1]));
        if (pair_any(bar, top > SLACK + BIAS || (m == NOTHING && top > -INFINITY))) {
          // raise the maxima to what they are, rescale l and O (each of the two threads half of its columns)
          half_max[half * RR + row] = top;
          pair_sync(bar);
          const float now = fmaxf(m, fmaxf(top, half_max[(half ^ 1) * RR + row]) - BIAS + ref), f = ex2(m - now);
          const float2 back = make_float2(ref - now, ref - now);
#pragma unroll
          for (int k = 0; k < 64; k += 2) {
            const float2 y = add2(make_float2(d[k], d[k + 1]), back);
            d[k] = y.x, d[k + 1] = y.y;
          }
          m = now;
          l *= f;
          if (j > 0) {
            wait_bar(&pdone[(tile - 1) & 1], ((tile - 1) >> 1) & 1, abort);
            __syncwarp();
            tc::fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 2; c += 16) {
              uint32_t o[16];
              tm_ld16(tlane + C::O + half * (HD / 2) + c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tm_st16(tlane + C::O + half * (HD / 2) + c, o);
            }
          }
        }
        const uint32_t to = tlane + C::P + tile % C::NP * C::PW + half * 48;
        uint32_t pa[16], pb[16], pc[16];
#pragma unroll
        for (int g = 0; g < 64 / GROUP; ++g) {
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int k = g * GROUP; k < (g + 1) * GROUP; k += 4) {
            const float2 x = make_float2(ex2(d[k]), ex2(d[k + 1])), y = make_float2(ex2(d[k + 2]), ex2(d[k + 3]));
            sum = add2(add2(x, y), sum);
            const __half2 hx = __floats2half2_rn(x.x, x.y), hy = __floats2half2_rn(y.x, y.y);
            uint32_t ax, bx, cx, ay, by, cy;
            split_weights<1>(hx, ax, bx, cx);
            split_weights<1>(hy, ay, by, cy);
            pa[k / 4] = upper_bytes(ax, ay);
            pb[k / 4] = upper_bytes(bx, by);
            pc[k / 4] = upper_bytes(cx, cy);
          }
          l = fmaf(sum.x + sum.y, s[g].z, l);
        }
        if (C::NP == 1 && j > 0) {
          wait_bar(&pdone[(tile - 1) & 1], ((tile - 1) >> 1) & 1, abort);
          __syncwarp();
          tc::fence_after();
        }
        tm_st16(to, pa);
        tm_st16(to + 16, pb);
        tm_st16(to + 32, pc);
        if (gaps && half == 0) {
          // a key that is not there: its value row is whatever lies in the slot, and 0·NaN is NaN
          wait_bar(&vfull[vslot], vturn, abort);
          if ((p.j0 + j) * TILE + row >= kv_end || s[row / GROUP].y == -INFINITY) {
            uint8_t* v = sV + vslot * C::SLOT + row * CW;
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
              for (int k = 0; k < CW / 16; ++k) *reinterpret_cast<uint4*>(v + cb * (TILE * CW) + k * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async_smem();
        }
        if (++vslot == NSV) {
          vslot = 0;
          vturn ^= 1u;
        }
        tm_wait_st();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&pfull[tile & 1]);
      }
    }
  }
  __syncthreads();
  if (*abort) {   // a wait ran out: give copies and products in flight time to land before the memory is given back
#pragma unroll 1
    for (int i = 0; i < 4096; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == W_MMA) tc::tmem_dealloc(tmem, C::COLS);
}

template <int HD>
static int launch_rows_t(const qsp_attn_kv8_layer& L, const CUtensorMap& mk, const CUtensorMap& mv, int box_rows, cudaStream_t st) {
  using C = RowsCfg<HD>;
  auto kern = rows_kernel<HD>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::BYTES);
  if (e != cudaSuccess) return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: %s", cudaGetErrorString(e));
  const int n_rg = (L.n_heads / L.n_kv_heads * L.tokens + RR - 1) / RR, G = grid_for(L, n_rg, TILE, tc::sm_count());
  const bool vec = aligned(L.qkv, 16) && aligned(L.out, 16) && L.ld_qkv % 8 == 0 && L.ld_out % 8 == 0;
  const int rc = launch_pdl("qsp_attn_kv8_verify(rows)", kern, dim3(G), dim3(C::THREADS), C::BYTES, st, mk, mv, L, n_rg, box_rows, vec);
  return rc ? rc : launch_merge(L, G, RR, TILE, st);
}

int launch_rows(const qsp_attn_kv8_layer& L, const CUtensorMap& mk, const CUtensorMap& mv, int box_rows, cudaStream_t st) {
  switch (L.head_dim) {
    case 32: return launch_rows_t<32>(L, mk, mv, box_rows, st);
    case 64: return launch_rows_t<64>(L, mk, mv, box_rows, st);
    case 128: return launch_rows_t<128>(L, mk, mv, box_rows, st);
    default: return launch_rows_t<256>(L, mk, mv, box_rows, st);
  }
}

int rows_error(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv8_error, sizeof(int));
  if (reset && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_kv8_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace kv8
}  // namespace qsp
