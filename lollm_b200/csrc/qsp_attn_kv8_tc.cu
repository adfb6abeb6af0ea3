// Attention over the 8-bit KV cache on tcgen05 tensor cores: bf16 models, page sizes that are a
// multiple of 8.
//
// The products read the codes as they lie in the cache: nothing is dequantised. The other operand
// is brought to 8 bits without losing what 16 bits hold, as the sum of two e4m3 values:
//   q·2^-e      = hi + lo/16   hi = e4m3(q·2^-e), lo = e4m3(16·(q·2^-e − hi)), 2^e a power of two per row
//   p·2^(v)     = hi + lo/16   of the softmax weights
// e4m3 has 4 significant bits, so hi takes the upper 4 of a bf16's 8 and lo the lower 4, exactly; a
// weight keeps 8 bits, as it would in bf16. hi and lo are columns of one product, whose halves
// are added in fp32. The power-of-two scales of the keys multiply the scores; those of the values join
// the softmax: with y = log2(e)·s + log2(vscale), weights w = 2^(y − m), m the running maximum of y,
// O = Σ w·vcode, l = Σ w / vscale. A weight's rounding is then relative to the largest contribution.
//
// Both products are transposed, so that the 128 rows of a tensor-core tile are keys (then head
// dims) and not the few query rows of a verify step:
//   S^T [128 keys, 2R]    = K [128, hd] · Q^T          A = the K tile, B = Q, hi rows then lo rows
//   O^T [hd, 2R]         += V^T [hd, 128] · P^T        A = the V tile read along its rows, B = P
// with R = 8..64 query rows (tokens × heads of the kv head). A thread of the softmax has one key
// and all R rows: its scales are scalars, the sum over keys is left to the end, and the maximum over
// keys need not be known exactly: m is raised (and O rescaled in TMEM) only when some score passes it
// by more than 2^SLACK; until then the check is one barrier with a vote.
//
// Warps: a softmax warpgroup for each 8 rows (R = 64: 16), two warps that load K and V (TMA), one that
// issues the MMAs. K and V tiles of 128 keys stream through a ring each, scores and weights are
// double-buffered, so the next tile's scores are computed while this one's weights are.
//
// Bound by HBM: a tile of 128 keys at hd 256 is 64 KB, 2800 cycles of an SM's share of 6.5 TB/s; its
// products take 520 cycles of the tensor cores at R = 32.
#include "qsp_attn_kv8.cuh"
#include "qsp_tc.cuh"

#include <algorithm>

namespace qsp {
namespace kv8 {

__device__ int g_kv8_error = 0;

constexpr int CODE_WAIT = 302;       // a bounded wait ran out
constexpr float SLACK = 2.f;         // log2 units the running maximum may lag behind
constexpr float BIAS = 6.f;          // weights are held times 2^BIAS: at most 2^(SLACK + BIAS) = 256 <= 448
constexpr float NOTHING = -1e30f;    // maximum of a row that has seen nothing

template <int HD, int R_>
struct Cfg {
  static constexpr int R = R_, N = 2 * R;                   // query rows, columns (hi | lo)
  static constexpr int NWG = R < 32 ? R / 8 : 4, RW = R / NWG;   // softmax warpgroups, rows of each
  static constexpr int CW = HD < 128 ? HD : 128;            // bytes of a swizzled row
  static constexpr int CB = HD / CW;                        // column blocks of a tile
  static constexpr int SLOT = TILE * HD;                    // bytes of a K or V tile
  static constexpr int QB = N * HD, PB = TILE * N;
  static constexpr int OCC = HD == 256 || R >= 32 ? 1 : 2;  // CTAs per SM
  static constexpr int BUDGET = OCC == 1 ? 232448 : 115712;
  // barriers, row scales, row maxima, reduction buffer
  static constexpr int SMALL = 8 * 28 + 4 * (R + 2 * R + 4 * R) + 16;
  static constexpr int FIT = (BUDGET - SMALL - 6 * 2 * TILE - QB - 2 * PB) / SLOT;
  static constexpr int NS = FIT < 8 ? FIT : 8;              // ring slots
  static constexpr int NSV = (NS + 1) / 2, NSK = NS - NSV;  // a V tile waits for its weights, a K tile does not
  static constexpr int NSE = NSK + 2;                       // slots of scale exponents
  static constexpr size_t BYTES = (size_t)NS * SLOT + QB + 2 * PB + SMALL + NSE * 2 * TILE;
  static constexpr int SOFTMAX = 128 * NWG, THREADS = SOFTMAX + 128;
  static constexpr int COLS_USED = 2 * N + CB * N;
  static constexpr int COLS = COLS_USED <= 64 ? 64 : COLS_USED <= 128 ? 128 : COLS_USED <= 256 ? 256 : 512;
  static_assert(NSK >= 2, "ring too short");
  static_assert(2 * PB >= 34 * 8, "the weights' buffers first hold share()'s 34 long longs");
};

// ---------------------------------------------------------------- descriptors
// rows of W bytes (16, 32, 64 or 128), swizzled over W bytes, 8-row groups 8·W apart: the layout of
// TMA boxes with inner extent W. K-major: rows are M/N, bytes along the row K. MN-major: the row is
// M/N, rows are K; lead = distance of the next W elements along M/N (0: the same again).
template <int W>
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lead) {
  constexpr uint64_t type = W == 128 ? 2 : W == 64 ? 4 : W == 32 ? 6 : 0;
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(8 * W >> 4) << 32 | 1ull << 46 | type << 61;
}
template <int W>
__device__ __forceinline__ int swz(int row, int chunk) {   // byte offset of a 16-byte chunk of a row
  constexpr int M = W / 16 - 1;
  return row * W + ((chunk ^ (row * W / 128 & M)) << 4);
}
// kind::f8f6f4, D fp32, A and B e4m3
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N, bool mn_major) {
  return (1u << 4) | (mn_major ? 3u << 15 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3_warp(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred e, p;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// ---------------------------------------------------------------- TMEM, n columns of this warp's 32 lanes
template <int N>
__device__ __forceinline__ void tm_ld(uint32_t t, uint32_t* r) {
  if constexpr (N == 32) {
    tm_ld<16>(t, r);
    tm_ld<16>(t + 16, r + 16);
  } else if constexpr (N == 16) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(t));
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(t));
  }
}
template <int N>
__device__ __forceinline__ void tm_st(uint32_t t, const uint32_t* r) {
  if constexpr (N > 8) {
    tm_st<N / 2>(t, r);
    tm_st<N / 2>(t + N / 2, r + N / 2);
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint16_t half2_to_e4m3x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<uint32_t*>(&v)));
  return r;
}
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

// v[RW] per lane -> in lane i the reduction over the warp's lanes of row row_of(i)
template <int RW, bool MAX>
__device__ __forceinline__ float warp_transpose_reduce(float (&v)[RW], int lane) {
  auto op = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  int o = 16;
#pragma unroll
  for (int n = RW / 2; n >= 1; n /= 2, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  float x = v[0];
#pragma unroll
  for (; o > 0; o >>= 1) x = op(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
template <int RW>
__device__ __forceinline__ int row_of(int lane) {
  return lane / (32 / RW);
}

constexpr uint32_t MISSING = 0xffffu;   // scale exponents of a key that has no page

template <int HD, int R_>
__global__ void __launch_bounds__(Cfg<HD, R_>::THREADS, Cfg<HD, R_>::OCC)
tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const qsp_attn_kv8_layer L, int n_rg,
          int box_rows) {
  using C = Cfg<HD, R_>;
  constexpr int R = C::R, N = C::N, RW = C::RW, NWG = C::NWG, NSK = C::NSK, NSV = C::NSV, CW = C::CW, CB = C::CB, EPL = HD / 32;
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t sK[];                // the swizzles go by address: 1024-byte tiles
  uint8_t* sV = sK + NSK * C::SLOT;
  uint8_t* sQ = sV + NSV * C::SLOT;
  uint8_t* sP = sQ + C::QB;                                      // [2][128 keys][N]
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sP + 2 * C::PB);
  uint64_t* kempty = kfull + NSK;
  uint64_t* vfull = kempty + NSK;
  uint64_t* vempty = vfull + NSV;
  uint64_t* sfull = vempty + NSV;  // scores of a tile are in TMEM
  uint64_t* sempty = sfull + 2;    // ... and have been read
  uint64_t* pfull = sempty + 2;    // weights of a tile are in shared memory
  uint64_t* pdone = pfull + 2;     // ... and their product with V is done
  uint64_t* qfull = pdone + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kfull + 27);   // after at most 2·8 + 9 barriers
  float* qs = reinterpret_cast<float*>(kfull + 28);   // [R] scale of a row's scores, in log2 units
  float* mcur = qs + R;                               // [R] running maximum
  float* aux = mcur + R;                              // [R] rescaling factor; 1 / l at the end
  float* red = aux + R;                               // [NWG][4][RW]
  volatile int* abort = reinterpret_cast<volatile int*>(red + 4 * R);
  uint16_t* sE = reinterpret_cast<uint16_t*>(red + 4 * R + 4);   // [NSE][128] a key's scale exponents + 127: K low, V high byte
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int W_K = 4 * NWG, W_V = W_K + 1, W_E = W_K + 2, W_MMA = W_K + 3;
  const int nrep = L.n_heads / L.n_kv_heads, rows_total = nrep * L.tokens;

  if (tid == 0) {
    for (int i = 0; i < 2 * C::NS; ++i) tc::mbar_init(&kfull[i], i < NSK ? 2 : 1);   // kfull (K and its scales), kempty, vfull, vempty
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sfull[i], 1);
      tc::mbar_init(&sempty[i], 4 * NWG);
      tc::mbar_init(&pfull[i], 4 * NWG);
      tc::mbar_init(&pdone[i], 1);
    }
    tc::mbar_init(qfull, 4 * NWG);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == W_MMA) {
    tc::tmem_alloc(tmem_slot, C::COLS);
    tc::fence_before();
  }
  pdl_wait();
  // the weights' buffers are not in use yet: room for share()'s 34 long longs
  Walk w = share(L, n_rg, R, reinterpret_cast<long long*>(sP));
  tc::fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const Scratch ws = scratch(L, gridDim.x, R);
  auto wait = [&](uint64_t* bar, uint32_t parity) { tc::mbar_wait(bar, parity, CODE_WAIT, &g_kv8_error, abort); };
  const int cap = L.max_pages * L.page_size;
  auto base_of = [&](int b) { return min(L.seq_lens[b], cap); };
  auto kv_end_of = [&](int base) { return min(base + L.tokens, cap); };   // keys that can have a page
  Piece p;
  p.n = 0;

  if (warp == W_K || warp == W_V) {
    // ---------------- loads of K and of V: up to 32 boxes a tile (box_rows keys x a column block each),
    // lane i looks up the page of box i, one tile ahead
    const bool is_v = warp == W_V;
    const CUtensorMap* map = is_v ? &tmV : &tmK;
    uint8_t* ring = is_v ? sV : sK;
    uint64_t* full = is_v ? vfull : kfull;
    uint64_t* empty = is_v ? vempty : kempty;
    const int slots = is_v ? NSV : NSK;
    const int chunks = TILE / box_rows, boxes = chunks * CB;
    int slot = 0;
    uint32_t turn = 1;   // parity of "empty" for this turn of the ring
    while (next_piece(L, n_rg, R, w, p)) {
      const int kv_end = kv_end_of(base_of(p.b));
      const int32_t* pages = L.page_table + (int64_t)p.b * L.max_pages;
      int key = p.j0 * TILE + lane % chunks * box_rows;
      auto page_at = [&](int j) { return j < p.n && lane < boxes && key < kv_end ? pages[key / L.page_size] : -1; };
      int page = page_at(0);
      for (int j = 0; j < p.n; ++j) {
        // row of the pages' [pages·n_kv·page_size, hd] view, or -1
        const int row = page >= 0 && page < L.num_pages ? (page * L.n_kv_heads + p.g) * L.page_size + key % L.page_size : -1;
        key += TILE;
        page = page_at(j + 1);
        wait(&empty[slot], turn);
        const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
        tc::mbar_expect_tx_warp(&full[slot], __popc(there) * box_rows * CW);
        uint8_t* dst = ring + slot * C::SLOT;
        for (int i = 0; i < boxes; ++i) {
          const int r = __shfl_sync(0xffffffffu, row, i);
          if (r >= 0) {
            const int cb = i / chunks;
            tc::tma_load_2d_warp(dst + cb * (TILE * CW) + (i - cb * chunks) * (box_rows * CW), map, &full[slot], cb * CW, r);
          }
        }
        if (++slot == slots) {
          slot = 0;
          turn ^= 1u;
        }
      }
    }
  } else if (warp == W_E) {
    // ---------------- scale exponents of a tile's keys, 4 a lane, in step with the K ring: pages are loaded two
    // tiles ahead, scales one. A slot is free when QK of the tile NSK before this one is done: that product was
    // issued after the scores of the tile NSE before, and so its scales, had been read.
    const int nb = L.page_size / L.scale_block, sb_log = __ffs(L.scale_block) - 1;
    uint32_t tile = 0;
    while (next_piece(L, n_rg, R, w, p)) {
      const int kv_end = kv_end_of(base_of(p.b));
      const int32_t* pages = L.page_table + (int64_t)p.b * L.max_pages;
      int page[4], slot[4];      // of tile j + 1, then j + 2
      float ks[4], vs[4];        // of tile j
      bool here[4];
      auto pages_at = [&](int j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = (p.j0 + j) * TILE + i * 32 + lane;
          const int lp = key / L.page_size;
          slot[i] = key - lp * L.page_size;
          page[i] = j < p.n && key < kv_end ? pages[lp] : -1;
        }
      };
      auto scales_at = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          here[i] = page[i] >= 0 && page[i] < L.num_pages;
          const int64_t at = here[i] ? ((int64_t)page[i] * L.n_kv_heads + p.g) * nb + (slot[i] >> sb_log) : 0;
          ks[i] = L.k_scales[at];
          vs[i] = L.v_scales[at];
        }
      };
      pages_at(0);
      scales_at();
      pages_at(1);
      for (int j = 0; j < p.n; ++j, ++tile) {
        const int s = tile % NSK;
        wait(&kempty[s], ((tile / NSK) & 1u) ^ 1u);
        uint16_t* e = sE + tile % C::NSE * TILE;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e[i * 32 + lane] = here[i] ? (uint16_t)((__float_as_uint(ks[i]) >> 23 & 0xffu) | (__float_as_uint(vs[i]) >> 23 & 0xffu) << 8)
                                     : (uint16_t)MISSING;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&kfull[s]);
        scales_at();
        pages_at(j + 2);
      }
    }
  } else if (warp == W_MMA) {
    // ---------------- products
    constexpr uint32_t ID_QK = idesc_e4m3(128, N, false), ID_PV = idesc_e4m3(128, N, true);
    uint32_t tile = 0, piece = 0;
    while (next_piece(L, n_rg, R, w, p)) {
      wait(qfull, piece & 1u);
      ++piece;
      const uint32_t t0 = tile;
      auto qk = [&](uint32_t t) {
        const int slot = t % NSK, sb = t & 1;
        wait(&kfull[slot], (t / NSK) & 1u);
        wait(&sempty[sb], ((t >> 1) & 1u) ^ 1u);
        tc::fence_after();
        const uint32_t a = tc::smem_u32(sK + slot * C::SLOT), q = tc::smem_u32(sQ);
#pragma unroll
        for (int k = 0; k < HD / 32; ++k) {
          const int cb = k * 32 / CW, off = k * 32 % CW;
          umma_e4m3_warp(tmem + sb * N, sdesc<CW>(a + cb * (TILE * CW) + off, 16), sdesc<CW>(q + cb * (N * CW) + off, 16), ID_QK, k > 0);
        }
        tc::umma_commit_warp(&kempty[slot]);
        tc::umma_commit_warp(&sfull[sb]);
      };
      auto pv = [&](uint32_t t) {
        const int slot = t % NSV, pb = t & 1;
        wait(&vfull[slot], (t / NSV) & 1u);
        wait(&pfull[pb], (t >> 1) & 1u);
        tc::fence_after();
        const uint32_t v = tc::smem_u32(sV + slot * C::SLOT), pp = tc::smem_u32(sP + pb * C::PB);
#pragma unroll
        for (int k = 0; k < TILE / 32; ++k) {
#pragma unroll
          for (int mb = 0; mb < CB; ++mb)
            umma_e4m3_warp(tmem + 2 * N + mb * N, sdesc<CW>(v + mb * (TILE * CW) + k * 32 * CW, 0),
                           N == 16 ? sdesc<16>(pp + k * 32 * N, 8 * 16) : sdesc<N < 32 ? 32 : N>(pp + k * 32 * N, 0), ID_PV,
                           t > t0 || k > 0);
        }
        tc::umma_commit_warp(&vempty[slot]);
        tc::umma_commit_warp(&pdone[pb]);
      };
      qk(t0);
      for (int j = 0; j < p.n; ++j) {
        if (j + 1 < p.n) qk(t0 + j + 1);
        pv(t0 + j);
      }
      tile = t0 + p.n;
    }
  } else {
    // ---------------- softmax: thread = key of the tile, RW rows
    const int wg = warp >> 2, wq = warp & 3, key_in = wq * 32 + lane, r0 = wg * RW, bar = 1 + wg;
    const uint32_t tlane = tmem + ((uint32_t)(wq * 32) << 16);
    const int my_row = r0 + row_of<RW>(lane);
    const bool reducer = lane % (32 / RW) == 0;    // its lane of a row's reduction
    uint32_t tile = 0;
    while (next_piece(L, n_rg, R, w, p)) {
      const int row0 = p.rg * R, nrows = min(R, rows_total - row0);
      const int base = base_of(p.b);
      const int key0 = p.j0 * TILE + key_in;

      // stage Q: a warp per row, hi at row r and lo at row R + r of the swizzled tile
      constexpr int ROWS = R / (4 * NWG);
      float x[ROWS][EPL];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = warp + i * 4 * NWG;
        if (r < nrows) {
          const int rr = row0 + r, t = rr / nrep, hq = p.g * nrep + rr - t * nrep;
          load_row<__nv_bfloat16, EPL>(
              static_cast<const __nv_bfloat16*>(L.q_buf) + (((int64_t)p.b * L.tokens + t) * L.n_heads + hq) * HD, lane, true, x[i]);
        } else {
#pragma unroll
          for (int k = 0; k < EPL; ++k) x[i][k] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = warp + i * 4 * NWG;
        float amax = 0.f;
        bool fine = true;
#pragma unroll
        for (int k = 0; k < EPL; ++k) {
          amax = fmaxf(amax, fabsf(x[i][k]));
          fine = fine && isfinite(x[i][k]);
        }
        amax = warp_max(amax);
        fine = __all_sync(0xffffffffu, fine);
        const int e = fine ? scale_exp(amax) : 0;
        const float inv = exp2i(-e);
        // pairs of codes, packed to the lane's EPL bytes
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < EPL; k += 2) {
          const float a = fine ? x[i][k] * inv : 0.f, z = fine && EPL > 1 ? x[i][EPL > 1 ? k + 1 : 0] * inv : 0.f;
          const uint16_t h = to_e4m3x2(a, z);
          const float2 f = from_e4m3x2(h);
          hi[k / 4] |= (uint32_t)h << (k % 4 * 8);
          lo[k / 4] |= (uint32_t)to_e4m3x2((a - f.x) * 16.f, (z - f.y) * 16.f) << (k % 4 * 8);
        }
        const int byte = lane * EPL, cb = byte / CW, in = byte % CW;
        store_bytes<EPL>(sQ + cb * (N * CW) + swz<CW>(r, in / 16) + in % 16, hi[0], hi[1]);
        store_bytes<EPL>(sQ + cb * (N * CW) + swz<CW>(R + r, in / 16) + in % 16, lo[0], lo[1]);
        if (lane == 0) {
          qs[r] = fine ? exp2i(e) * (L.scale * LOG2E) : NAN;
          mcur[r] = NOTHING;
        }
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(qfull);
      asm volatile("barrier.cta.sync 15, %0;" ::"n"(C::SOFTMAX) : "memory");   // qs and mcur of all rows are written

      float m[RW], l[RW], qr[RW == 8 ? 8 : 1];
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        m[i] = NOTHING;
        l[i] = 0.f;
        if (RW == 8) qr[i] = qs[r0 + i];
      }
      auto q_scale = [&](int i) { return RW == 8 ? qr[i] : qs[r0 + i]; };   // 16 rows: registers are short
      // last key that the first of all rows of this warpgroup sees
      const int seen_by_all = base + (row0 + r0) / nrep;

      for (int j = 0; j < p.n; ++j, ++tile) {
        const uint32_t sb = tile & 1, ph = (tile >> 1) & 1;
        const int key = key0 + j * TILE;
        wait(&sfull[sb], ph);
        tc::fence_after();
        uint32_t ev = sE[tile % C::NSE * TILE + key_in];
        const bool mine = ev != MISSING;   // the key exists
        if (!mine) ev = 127u << 8 | 127u;
        const float ks = __uint_as_float((ev & 0xffu) << 23);
        const float ve = (float)(int)(ev >> 8) - (127.f - BIAS), ivs = exp2i(127 - max((int)(ev >> 8), 1));
        // rows that may see this key: all, but for missing keys and the tiles of the new tokens
        uint32_t sees = mine ? 0xffffffffu : 0u;
        if (mine && key > seen_by_all) {
#pragma unroll
          for (int i = 1; i < RW; ++i)
            if (key > base + (row0 + r0 + i) / nrep) sees &= ~(1u << i);
          sees &= ~1u;
        }
        uint32_t sh[RW], sl[RW];
        tm_ld<RW>(tlane + sb * N + r0, sh);
        tm_ld<RW>(tlane + sb * N + R + r0, sl);
        tm_wait_ld();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sempty[sb]);

        // d: exponents of the weights; scores times qr·ks are in log2 units
        float x[RW], d[RW];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
          x[i] = fmaf(__uint_as_float(sl[i]), 0.0625f, __uint_as_float(sh[i]));
          d[i] = fmaf(x[i], q_scale(i) * ks, ve - m[i]);
        }
        if (sees != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < RW; ++i)
            if (!(sees >> i & 1)) d[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) top = fmaxf(top, d[i]);
        if (bar_any(bar, top > SLACK + BIAS)) {
          // raise the maxima to what they are, rescale l and O
          float y[RW];
#pragma unroll
          for (int i = 0; i < RW; ++i) y[i] = sees >> i & 1 ? fmaf(x[i], q_scale(i) * ks, ve - BIAS) : -INFINITY;
          const float best = warp_transpose_reduce<RW, true>(y, lane);
          if (reducer) red[wg * 4 * RW + row_of<RW>(lane) * 4 + wq] = best;
          bar_sync(bar);
          if (wq == 0 && reducer) {
            const float4 v = *reinterpret_cast<const float4*>(red + wg * 4 * RW + row_of<RW>(lane) * 4);
            const float was = mcur[my_row];
            const float now = fmaxf(was, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
            mcur[my_row] = now;
            aux[my_row] = ex2(was - now);
          }
          bar_sync(bar);
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            m[i] = mcur[r0 + i];
            l[i] *= aux[r0 + i];
            d[i] = sees >> i & 1 ? fmaf(x[i], q_scale(i) * ks, ve - m[i]) : -INFINITY;
          }
          if (j > 0) {
            const uint32_t t1 = tile - 1;
            wait(&pdone[t1 & 1], (t1 >> 1) & 1);
            tc::fence_after();
#pragma unroll 1
            for (int c = 0; c < CB * 2; ++c) {
              uint32_t o[RW];
              const uint32_t where = tlane + 2 * N + (c >> 1) * N + (c & 1) * R + r0;
              tm_ld<RW>(where, o);
              tm_wait_ld();
#pragma unroll
              for (int i = 0; i < RW; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * aux[r0 + i]);
              tm_st<RW>(where, o);
            }
            tm_wait_st();
            tc::fence_before();
          }
        }
        // weights, as two e4m3 values each
        uint32_t hi[RW / 4], lo[RW / 4];
#pragma unroll
        for (int i = 0; i < RW; i += 2) {
          const float a = ex2(d[i]), z = ex2(d[i + 1]);
          l[i] = fmaf(a, ivs, l[i]);
          l[i + 1] = fmaf(z, ivs, l[i + 1]);
          const __half2 wv = __floats2half2_rn(a, z);
          const uint16_t h = half2_to_e4m3x2(wv);
          const uint16_t q = half2_to_e4m3x2(__hmul2(__hsub2(wv, e4m3x2_to_half2(h)), __float2half2_rn(16.f)));
          if (i % 4 == 0) {
            hi[i / 4] = h;
            lo[i / 4] = q;
          } else {
            hi[i / 4] |= (uint32_t)h << 16;
            lo[i / 4] |= (uint32_t)q << 16;
          }
        }
        // (the buffer's previous product, of tile - 2, was issued before QK of this tile and so is done)
        uint8_t* pr = sP + sb * C::PB;
        if constexpr (R == 8) {
          *reinterpret_cast<uint4*>(pr + key_in * 16) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
        } else if constexpr (RW == 8) {
          *reinterpret_cast<uint2*>(pr + swz<N>(key_in, r0 / 16) + r0 % 16) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(pr + swz<N>(key_in, (R + r0) / 16) + r0 % 16) = make_uint2(lo[0], lo[1]);
        } else {
          *reinterpret_cast<uint4*>(pr + swz<N>(key_in, r0 / 16)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(pr + swz<N>(key_in, (R + r0) / 16)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (!mine && wg == 0) {
          // a key that is not there: its value row is whatever lies in the slot, and 0·NaN is NaN
          wait(&vfull[tile % NSV], (tile / NSV) & 1u);
          uint8_t* v = sV + tile % NSV * C::SLOT + key_in * CW;
#pragma unroll
          for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int k = 0; k < CW / 16; ++k) *reinterpret_cast<uint4*>(v + cb * (TILE * CW) + k * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&pfull[sb]);
      }

      // ---- the piece is done: l over the keys, O out of TMEM (thread = head dim)
      const float s = warp_transpose_reduce<RW, false>(l, lane);
      if (reducer) red[wg * 4 * RW + row_of<RW>(lane) * 4 + wq] = s;
      const uint32_t t1 = tile - 1;
      wait(&pdone[t1 & 1], (t1 >> 1) & 1);
      tc::fence_after();
      bar_sync(bar);
      const bool whole = p.whole();
      if (wq == 0 && reducer) {
        const float4 v4 = *reinterpret_cast<const float4*>(red + wg * 4 * RW + row_of<RW>(lane) * 4);
        const float v = (v4.x + v4.y) + (v4.z + v4.w);
        aux[my_row] = v == 0.f ? 0.f : 1.f / v;
        if (!whole) ws.ml[(int64_t)p.slot() * R + my_row] = make_float2(v == 0.f ? -INFINITY : mcur[my_row], v);
      }
      bar_sync(bar);
#pragma unroll 1
      for (int mb = 0; mb < CB; ++mb) {
        uint32_t oh[RW], ol[RW];
        tm_ld<RW>(tlane + 2 * N + mb * N + r0, oh);
        tm_ld<RW>(tlane + 2 * N + mb * N + R + r0, ol);
        tm_wait_ld();
        const int dim = mb * 128 + key_in;
        if (dim < HD) {
          if (whole) {
#pragma unroll
            for (int i = 0; i < RW; ++i) {
              if (r0 + i < nrows) {
                const int rr = row0 + r0 + i, t = rr / nrep, hq = p.g * nrep + rr - t * nrep;
                const int64_t mrow = (int64_t)p.b * L.tokens + t;
                const float gate = __bfloat162float(static_cast<const __nv_bfloat16*>(L.qkv)[mrow * L.ld_qkv + (int64_t)hq * 2 * HD + HD + dim]);
                const float o = fmaf(__uint_as_float(ol[i]), 0.0625f, __uint_as_float(oh[i])) * aux[r0 + i];
                static_cast<__nv_bfloat16*>(L.out)[mrow * L.ld_out + (int64_t)hq * HD + dim] = __float2bfloat16_rn(o * sigmoidf_(gate));
              }
            }
          } else {
            float* o = ws.o + ((int64_t)p.slot() * R + r0) * HD + dim;
#pragma unroll
            for (int i = 0; i < RW; ++i) o[i * HD] = fmaf(__uint_as_float(ol[i]), 0.0625f, __uint_as_float(oh[i]));
          }
        }
      }
      tc::fence_before();   // the next piece's products overwrite O after its pfull
      asm volatile("barrier.cta.sync 15, %0;" ::"n"(C::SOFTMAX) : "memory");   // qs, mcur, aux are written again
    }
    if (tid == 0) put_meta(ws, w, p);
  }
  __syncthreads();
  if (*abort) {   // a wait ran out: give copies and products in flight time to land before the memory is given back
    for (int i = 0; i < 4096; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == W_MMA) tc::tmem_dealloc(tmem, C::COLS);
}

// [pages·n_kv·page_size rows, hd] codes, box of box_rows x CW bytes swizzled over CW
static bool make_map(CUtensorMap* m, const void* base, int64_t rows, int hd, int box_rows) {
  tc::EncodeTiled enc = tc::get_encode();
  if (!enc) return false;
  const int cw = std::min(hd, 128);
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)hd};
  cuuint32_t box[2] = {(cuuint32_t)cw, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1, 1};
  const CUtensorMapSwizzle sw = cw == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : cw == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int tc_grid(int hd, int R) { return tc::sm_count() * (hd == 256 || R >= 32 ? 1 : 2); }

// the least R that holds all query rows of a kv head, so that each key is read once; 64 at most
int tc_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

template <int HD, int R>
static int launch_tc_t(const qsp_attn_kv8_layer& L, cudaStream_t st) {
  using C = Cfg<HD, R>;
  const int64_t rows = (int64_t)L.num_pages * L.n_kv_heads * L.page_size;
  int box_rows = 8;
  while (box_rows < TILE && L.page_size % (2 * box_rows) == 0) box_rows *= 2;
  CUtensorMap mk, mv;
  if (!make_map(&mk, L.k_pages, rows, HD, box_rows) || !make_map(&mv, L.v_pages, rows, HD, box_rows))
    return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: no tensor map for the pages");
  auto kern = tc_kernel<HD, R>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::BYTES);
  if (e != cudaSuccess) return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: %s", cudaGetErrorString(e));
  const int G = tc_grid(HD, R), n_rg = (L.n_heads / L.n_kv_heads * L.tokens + R - 1) / R;
  const int rc = launch_pdl("qsp_attn_kv8_verify", kern, dim3(G), dim3(C::THREADS), C::BYTES, st, mk, mv, L, n_rg, box_rows);
  return rc ? rc : launch_merge(L, G, R, st);
}

template <int HD>
static int launch_tc_hd(const qsp_attn_kv8_layer& L, cudaStream_t st) {
  switch (tc_rows(L.n_heads / L.n_kv_heads * L.tokens)) {
    case 8: return launch_tc_t<HD, 8>(L, st);
    case 16: return launch_tc_t<HD, 16>(L, st);
    case 32: return launch_tc_t<HD, 32>(L, st);
    default: return launch_tc_t<HD, 64>(L, st);
  }
}

int launch_tc(const qsp_attn_kv8_layer& L, cudaStream_t st) {
  // rows of the pages are 32-bit coordinates of the tensor map
  if (L.page_size % 8 != 0 || (int64_t)L.num_pages * L.n_kv_heads * L.page_size >= (1ll << 31)) return QSP_ERR_UNSUPPORTED;
  switch (L.head_dim) {
    case 32: return launch_tc_hd<32>(L, st);
    case 64: return launch_tc_hd<64>(L, st);
    case 128: return launch_tc_hd<128>(L, st);
    default: return launch_tc_hd<256>(L, st);
  }
}

int device_error(int reset) {
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
