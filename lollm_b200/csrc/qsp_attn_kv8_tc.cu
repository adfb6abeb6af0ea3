// Attention over the 8-bit KV cache on tcgen05 tensor cores: bf16 models, page sizes that are a
// multiple of 8. tc_kernel, here, takes up to 64 query rows of a kv head (tokens x heads) and any number of
// them in groups of 64; chunks of prompts have a kernel of their own, with 128 (rows_kernel).
//
// The products read the codes as they lie in the cache: nothing is dequantised. The other operand
// is brought to 8 bits as a sum:
//   q·2^-e      = hi + lo/16        hi = e4m3(q·2^-e), lo = e4m3(16·(q·2^-e − hi)), 2^e a power of two per row
//   p·2^(v)     = a + (b + c)/4     e5m2, of the softmax weights (split_weights)
// e4m3 has 4 significant bits, so hi takes the upper 4 of a bf16's 8 and lo the lower 4: exactly for elements down to
// 2^-6, of a row whose largest is scaled to 224..448; smaller ones are off by at most 2^-14, 2^-21 of the largest. A weight
// has the precision of bf16 down to 2^-22 of the row's largest. hi and lo, a and b are columns of one product,
// whose halves are added in fp32; c is a product of its own into b's columns, since TMEM has no more for a third
// part of 64 rows. The power-of-two scales of the keys multiply the scores; those of the values join
// the softmax: with y = log2(e)·s + log2(vscale), weights w = 2^(y − m), m the running maximum of y,
// O = Σ w·vcode, l = Σ w / vscale. A weight's rounding is then relative to the largest contribution.
//
// Both products are transposed, so that the 128 rows of a tensor-core tile are keys (then head
// dims) and not the few query rows of a verify step:
//   S^T [128 keys, 2R]    = K [128, hd] · Q^T          A = the K tile, B = Q, hi rows then lo rows
//   O^T [hd, 2R]         += V^T [hd, 128] · P^T        A = the V tile read along its rows, B = P, a rows then b rows
//   O^T [hd, second R]   += V^T [hd, 128] · Pc^T       B = the weights' c rows
// with R = 8..64 query rows (tokens × heads of the kv head). A thread of the softmax has one key
// and all R rows: its scales are scalars, the sum over keys is left to the end, and the maximum over
// keys need not be known exactly: m is raised (and O rescaled in TMEM) only when some score passes it
// by more than 2^SLACK; until then the check is one barrier with a vote.
//
// Warps: a softmax warpgroup for each 8 rows (R = 64: 16), a warp each that loads K, loads V (TMA), brings the
// scales (and walks through the work), issues the MMAs. K and V tiles of 128 keys stream through a ring each,
// scores and weights are double-buffered, so the next tile's scores are computed while this one's weights are.
//
// Bound by HBM where sequences are long: a tile of 128 keys at hd 256 is 64 KB, 2800 cycles of an SM's share of
// 6.5 TB/s; its products take 780 cycles of the tensor cores at R = 32, its softmax a chain of some 1900 cycles.
// Measured, 2 kv heads of 256, 64 sequences of 1k to 32k keys, 4 tokens: 174 us in a graph on one input, 210 (5.3 TB/s)
// on inputs that change (197 with weights of two parts); of 2048 to 2560 keys: 4 tokens 35 us in a graph, 38 on inputs that
// change (34, 36), 8 tokens (R = 64) 46 us (43). One token over 33 keys: 6.8 us, a chain of length, plan, page, scales and K, product, softmax, product, gate.
#include "qsp_attn_kv8_tc.cuh"

#include <algorithm>

namespace qsp {
namespace kv8 {

template <int HD, int R_>
struct Cfg {
  static constexpr int R = R_, N = 2 * R;                   // query rows, columns (hi | lo)
  static constexpr int NWG = R < 32 ? R / 8 : 4, RW = R / NWG;   // softmax warpgroups, rows of each
  static constexpr int CW = HD < 128 ? HD : 128;            // bytes of a swizzled row
  static constexpr int CB = HD / CW;                        // column blocks of a tile
  static constexpr int SLOT = TILE * HD;                    // bytes of a K or V tile
  static constexpr int NC = R < 16 ? 16 : R;                // columns of the weights' third part: an MMA has 16 at least
  static constexpr int QB = N * HD, PB = TILE * N, PCB = TILE * NC;
  static constexpr int OCC = HD == 256 || R >= 32 ? 1 : 2;  // CTAs per SM
  static constexpr size_t BUDGET = OCC == 1 ? 232448 : 115712;
  // barriers, piece descriptors, row scales (of two pieces), maxima and factors, reduction buffer
  static constexpr int SMALL = 8 * 34 + NDESC * 32 + 4 * (2 * R + 2 * R + 4 * R) + 16;
  // slots of scale exponents: two more than of K
  static constexpr size_t bytes(int ns) { return (size_t)ns * SLOT + QB + 2 * PB + 2 * PCB + SMALL + (ns / 2 + 2) * 2 * TILE; }
  static constexpr int slots() {
    int ns = 8;
    while (bytes(ns) > BUDGET) --ns;
    return ns;
  }
  static constexpr int NS = slots();                        // ring slots
  static constexpr int NSK = NS / 2, NSV = NS - NSK;        // a V tile waits for its weights, a K tile does not
  static constexpr int NSE = NSK + 2;
  static constexpr size_t BYTES = bytes(NS);
  static constexpr int SOFTMAX = 128 * NWG, THREADS = SOFTMAX + 128;
  static constexpr int COLS_USED = 2 * N + CB * N;
  static constexpr int COLS = COLS_USED <= 64 ? 64 : COLS_USED <= 128 ? 128 : COLS_USED <= 256 ? 256 : 512;
  static_assert(NSK >= 2 && NSK <= 4, "ring too short, or too long for the descriptors' slots");
  static_assert(2 * PB >= 68 * 4, "the weights' buffers first hold share()'s 68 ints");
};

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

template <int HD, int R_>
__global__ void __launch_bounds__(Cfg<HD, R_>::THREADS, Cfg<HD, R_>::OCC)
tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const qsp_attn_kv8_layer L, int n_rg,
          int box_rows) {
  using C = Cfg<HD, R_>;
  constexpr int R = C::R, N = C::N, NC = C::NC, RW = C::RW, NWG = C::NWG, NSK = C::NSK, NSV = C::NSV, CW = C::CW, CB = C::CB, EPL = HD / 32;
  extern __shared__ __align__(1024) uint8_t sK[];                // the swizzles go by address: 1024-byte tiles
  uint8_t* sV = sK + NSK * C::SLOT;
  uint8_t* sQ = sV + NSV * C::SLOT;
  uint8_t* sP = sQ + C::QB;                                      // [2][128 keys][N]
  uint8_t* sPc = sP + 2 * C::PB;                                 // [2][128 keys][NC]
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sPc + 2 * C::PCB);
  uint64_t* kempty = kfull + NSK;
  uint64_t* vfull = kempty + NSK;
  uint64_t* vempty = vfull + NSV;
  uint64_t* sfull = vempty + NSV;  // scores of a tile are in TMEM
  uint64_t* pfull = sfull + 2;     // weights of a tile are in shared memory (and its scores have been read)
  uint64_t* pdone = pfull + 2;     // ... and their product with V is done
  uint64_t* qfull = pdone + 2;     // Q of a piece is in shared memory
  uint64_t* dfull = qfull + 1;     // [NDESC] a piece's descriptor is there; 2·8 + 7 + 8 barriers at most
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kfull + 33);
  Desc* desc = reinterpret_cast<Desc*>(kfull + 34);
  float* qs = reinterpret_cast<float*>(desc + NDESC);   // [2][R] scale of a row's scores, in log2 units, by piece
  float* mcur = qs + 2 * R;                           // [R] running maximum
  float* aux = mcur + R;                              // [R] rescaling factor; 1 / l at the end
  float* red = aux + R;                               // [NWG][RW][4]
  volatile int* abort = reinterpret_cast<volatile int*>(red + 4 * R);
  uint16_t* sE = reinterpret_cast<uint16_t*>(red + 4 * R + 4);   // [NSE][128] a key's scale exponents + 127: K low, V high byte
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int W_K = 4 * NWG, W_V = W_K + 1, W_E = W_K + 2, W_MMA = W_K + 3;
  const int nrep = L.n_heads / L.n_kv_heads, rows_total = nrep * L.tokens;

  if (tid == 0) {
    for (int i = 0; i < 2 * C::NS; ++i) tc::mbar_init(&kfull[i], i < NSK ? 2 : 1);   // kfull (K and its scales), kempty, vfull, vempty
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sfull[i], 1);
      tc::mbar_init(&pfull[i], 4 * NWG);
      tc::mbar_init(&pdone[i], 1);
    }
    tc::mbar_init(qfull, 4 * NWG);
    for (int i = 0; i < NDESC; ++i) tc::mbar_init(&dfull[i], 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < R) mcur[tid] = NOTHING;
  if (lane == 0 && (warp == W_K || warp == W_V))
    asm volatile("prefetch.tensormap [%0];" ::"l"(warp == W_K ? &tmK : &tmV) : "memory");
  pdl_wait();
  // TMEM is asked for when the previous kernel has given its own back, and the next kernel may start when this
  // grid has all of its: a CTA that waits for a grid never holds columns that the grid's CTAs still need
  if (warp == W_MMA) {
    tc::tmem_alloc(tmem_slot, C::COLS);
    tc::fence_before();
  }
  // the weights' buffers are not in use yet: room for share()'s 68 ints
  Walk w = share<TILE>(L, n_rg, R, reinterpret_cast<int*>(sP));
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
    // ---------------- scale exponents of a tile's keys, 4 a lane
    uint16_t* e = sE + lane;
    const Piece p = walk_and_scales(L, n_rg, R, NSK, w, desc, dfull, kfull, kempty, abort, [&](const Scales& x) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        e[i * 32] = x.here[i] ? (uint16_t)((__float_as_uint(x.ks[i]) >> 23 & 0xffu) | (__float_as_uint(x.vs[i]) >> 23 & 0xffu) << 8)
                              : (uint16_t)MISSING;
      e += TILE;
      if (e == sE + lane + C::NSE * TILE) e = sE + lane;
    });
    if (lane == 0) put_meta(scratch(L, gridDim.x, R), w, p);
  } else if (warp == W_MMA) {
    // ---------------- products, in the order QK(0) QK(1) PV(0) QK(2) PV(1) ... of each piece. QK(t) overwrites the
    // scores of t - 2, which had been read when pfull(t - 2) came, before PV(t - 2) and so before QK(t).
    constexpr uint32_t ID_QK = idesc_f8(128, N, false, false), ID_PV = idesc_f8(128, N, true, true), ID_PC = idesc_f8(128, NC, true, true);
    const Sdesc dK = sdesc<CW>(sK, 16), dV = sdesc<CW>(sV, 0), dQ = sdesc<CW>(sQ, 16);
    const Sdesc dP = N == 16 ? sdesc<16>(sP, 8 * 16) : sdesc<N < 32 ? 32 : N>(sP, 0);
    const Sdesc dPc = NC == 16 ? sdesc<16>(sPc, 8 * 16) : sdesc<NC < 32 ? 32 : NC>(sPc, 0);
    uint32_t tile = 0, piece = 0, kslot = 0, kturn = 0, vslot = 0, vturn = 0;
    for (;; ++piece) {
      const int n = piece_at(piece).n;
      if (n == 0) break;
      wait_bar(qfull, piece & 1u, abort);
      auto qk = [&](uint32_t t) {
        const uint32_t sb = t & 1;
        wait_bar(&kfull[kslot], kturn, abort);
        __syncwarp();
        tc::fence_after();
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
          umma_f8_warp<CW / 32, 2, 2>(tmem + sb * N, {dK.lo + (kslot * C::SLOT + cb * (TILE * CW)) / 16, dK.hi},
                                        {dQ.lo + cb * (N * CW) / 16, dQ.hi}, ID_QK, cb > 0);
        tc::umma_commit_warp(&kempty[kslot]);
        tc::umma_commit_warp(&sfull[sb]);
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
        {
          const Sdesc v = {dV.lo + (vslot * C::SLOT + mb * (TILE * CW)) / 16, dV.hi};
          umma_f8_warp<4, 32 * CW / 16, 32 * N / 16>(tmem + 2 * N + mb * N, v, {dP.lo + pb * C::PB / 16, dP.hi}, ID_PV, j > 0);
          // (R = 8: zeros for a's columns)
          umma_f8_warp<4, 32 * CW / 16, 32 * NC / 16>(tmem + 2 * N + mb * N + N - NC, v, {dPc.lo + pb * C::PCB / 16, dPc.hi}, ID_PC, 1);
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
    // ---------------- softmax: thread = key of the tile, RW rows. Row r of the unit is column
    // (r / RW)·2RW + r % RW of the scores (hi), and RW columns further (lo): a warpgroup's are together. It is
    // columns r and R + r of the outputs.
    const int wg = warp >> 2, wq = warp & 3, key_in = wq * 32 + lane, r0 = wg * RW, bar = 1 + wg;
    const uint32_t tlane = tmem + ((uint32_t)(wq * 32) << 16) + wg * (2 * RW), tout = tmem + ((uint32_t)(wq * 32) << 16) + 2 * N + r0;
    const int my_row = r0 + row_of<RW>(lane);
    const bool reducer = lane % (32 / RW) == 0;    // its lane of a row's reduction
    const Scratch ws = scratch(L, gridDim.x, R);
    uint32_t tile = 0, piece = 0, eslot = 0, vslot = 0, vturn = 0;

    // Q of a piece: a warp per row, loaded one tile before it is staged (4 rows: when it is; registers are short)
    constexpr int ROWS = R / (4 * NWG);
    constexpr bool AHEAD = ROWS <= 2;
    Row<__nv_bfloat16, EPL> q_raw[ROWS];
    auto load_q = [&](const Desc& q) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int rr = q.row0 + warp + i * 4 * NWG;
        if (rr < rows_total) {
          const int t = rr / nrep, hq = q.g * nrep + rr - t * nrep;
          q_raw[i].load(static_cast<const __nv_bfloat16*>(L.q_buf) + (((int64_t)q.b * L.tokens + t) * L.n_heads + hq) * HD, lane, true);
        } else {
          q_raw[i].zero();
        }
      }
    };
    auto stage_q = [&](uint32_t n) {   // for the n-th piece
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = warp + i * 4 * NWG, row = r / RW * (2 * RW) + r % RW;
        const uint32_t top = __reduce_max_sync(0xffffffffu, q_raw[i].top());
        const bool fine = top < NOT_FINITE;
        const int e = fine ? scale_exp(top) : 0;
        const float inv = exp2i(-e);
        // pairs of codes, packed to the lane's EPL bytes
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < EPL; k += 2) {
          const float a = fine ? q_raw[i][k] * inv : 0.f, z = fine && EPL > 1 ? q_raw[i][EPL > 1 ? k + 1 : 0] * inv : 0.f;
          const uint16_t h = to_e4m3x2(a, z);
          const float2 f = from_e4m3x2(h);
          hi[k / 4] |= (uint32_t)h << (k % 4 * 8);
          lo[k / 4] |= (uint32_t)to_e4m3x2((a - f.x) * 16.f, (z - f.y) * 16.f) << (k % 4 * 8);
        }
        const int byte = lane * EPL, cb = byte / CW, in = byte % CW;
        store_bytes<EPL>(sQ + cb * (N * CW) + swz<CW>(row, in / 16) + in % 16, hi[0], hi[1]);
        store_bytes<EPL>(sQ + cb * (N * CW) + swz<CW>(row + RW, in / 16) + in % 16, lo[0], lo[1]);
        if (lane == 0) qs[(n & 1) * R + r] = fine ? exp2i(e) * (L.scale * LOG2E) : NAN;
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(qfull);
    };

    // the warps of a group meet at its barriers, so they have to agree on the next piece (they do, but for a
    // wait that ran out in one of them)
    auto agreed_piece_at = [&](uint32_t i) -> Desc {
      Desc d = piece_at(i);
      if (bar_any(bar, d.n == 0)) d.n = 0;
      return d;
    };
    Desc p = agreed_piece_at(0);
    if (p.n > 0) {
      load_q(p);
      stage_q(0);
    }
    while (p.n > 0) {
      const int row0 = p.row0 + r0;   // this warpgroup's first row
      const float* q_scale = qs + (piece & 1) * R + r0;
      const float* m = mcur + r0;     // shared memory: registers are short
      // token and head (in the group) of the first row; later rows follow by counting
      const int t_first = row0 / nrep, h_first = row0 - t_first * nrep;
      int key = p.j0 * TILE + key_in;
      bool more = false;

      float l[RW];
#pragma unroll
      for (int i = 0; i < RW; ++i) l[i] = 0.f;
      for (int j = 0; j < p.n; ++j, ++tile, key += TILE) {
        const uint32_t sb = tile & 1, ph = (tile >> 1) & 1;
        if (j == p.n - 1) {
          const Desc next = piece_at(piece + 1);
          more = next.n > 0;
          if (AHEAD && more) load_q(next);
          if (p.whole && wq == 0) {   // gates of this group's rows into L2: a quarter of a row a lane
#pragma unroll
            for (int i = 0; i < RW; i += 8) {
              const int rr = row0 + i + lane / 4, t = rr / nrep;
              if (rr < rows_total)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const __nv_bfloat16*>(L.qkv) + ((int64_t)p.b * L.tokens + t) * L.ld_qkv +
                                                               (int64_t)(p.g * nrep + rr - t * nrep) * 2 * HD + HD + lane % 4 * (HD / 4)));
            }
          }
        }
        wait_bar(&sfull[sb], ph, abort);
        __syncwarp();
        tc::fence_after();
        uint32_t ev = sE[eslot * TILE + key_in];
        if (++eslot == C::NSE) eslot = 0;
        const bool mine = ev != MISSING;   // the key exists
        if (!mine) ev = 127u << 8 | 127u;
        const float ks = __uint_as_float((ev & 0xffu) << 23);
        const float ve = (float)(int)(ev >> 8) - (127.f - BIAS), ivs = exp2i(127 - max((int)(ev >> 8), 1));
        // rows that may see this key: all, but for missing keys and the tiles of the new tokens
        uint32_t sees = mine ? 0xffffffffu : 0u;
        if (mine && key > p.base + t_first) {
          sees = 0;
          int t = p.base + t_first, h = h_first;
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            if (key <= t) sees |= 1u << i;
            if (++h == nrep) {
              h = 0;
              ++t;
            }
          }
        }
        const bool all = sees == 0xffffffffu;

        // d: exponents of the weights; scores times q_scale·ks are in log2 units
        auto exponents = [&](float (&d)[RW], bool over_max) {   // relative to the running maximum, or as they are
#pragma unroll
          for (int i = 0; i < RW; i += 8) {
            uint32_t hi[8], lo[8];
            tm_ld8(tlane + sb * N + i, hi);
            tm_ld8(tlane + sb * N + RW + i, lo);
            tm_wait_ld8(hi, lo);
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
              const float4 q = *reinterpret_cast<const float4*>(q_scale + i + k), mm = *reinterpret_cast<const float4*>(m + i + k);
              const float qq[4] = {q.x, q.y, q.z, q.w}, m4[4] = {mm.x, mm.y, mm.z, mm.w};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const float x = fmaf(__uint_as_float(lo[k + u]), 0.0625f, __uint_as_float(hi[k + u]));
                d[i + k + u] = fmaf(x, qq[u] * ks, over_max ? ve - m4[u] : ve - BIAS);
              }
            }
          }
          if (!all) {
#pragma unroll
            for (int i = 0; i < RW; ++i)
              if (!(sees >> i & 1)) d[i] = -INFINITY;
          }
        };
        float d[RW], top = -INFINITY;
        exponents(d, true);
#pragma unroll
        for (int i = 0; i < RW; ++i) top = fmaxf(top, d[i]);
        if (bar_any(bar, top > SLACK + BIAS)) {
          // raise the maxima to what they are, rescale l and O. (The scores are still in TMEM: until pfull.)
          exponents(d, false);
          const float best = warp_transpose_reduce<RW, true>(d, lane);
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
          exponents(d, true);
#pragma unroll
          for (int i = 0; i < RW; ++i) l[i] *= aux[r0 + i];
          if (j > 0) {
            wait_bar(&pdone[sb ^ 1], ((tile - 1) >> 1) & 1, abort);
            __syncwarp();
            tc::fence_after();
#pragma unroll 1
            for (int c = 0; c < CB * (RW / 4); ++c) {   // 8 columns
              const int mb = c / (RW / 4), i0 = c % (RW / 4) * 8;
              uint32_t o[8];
              const uint32_t where = tout + mb * N + i0 / RW * R + i0 % RW;
              tm_ld8(where, o);
              tm_wait_ld8(o);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * aux[r0 + i0 % RW + i]);
              tm_st8(where, o);
            }
            tm_wait_st();
            tc::fence_before();
          }
        }
        // weights, as three e5m2 values each. (The buffer's previous product, of tile - 2, was issued before QK of
        // this tile and so is done.)
        uint32_t pa[RW / 4], pb[RW / 4], pc[RW / 4];
#pragma unroll
        for (int i = 0; i < RW; i += 4) {
          uint32_t x[2][3];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float a = ex2(d[i + 2 * k]), z = ex2(d[i + 2 * k + 1]);
            l[i + 2 * k] = fmaf(a, ivs, l[i + 2 * k]);
            l[i + 2 * k + 1] = fmaf(z, ivs, l[i + 2 * k + 1]);
            split_weights<4>(__floats2half2_rn(a, z), x[k][0], x[k][1], x[k][2]);
          }
          pa[i / 4] = upper_bytes(x[0][0], x[1][0]);
          pb[i / 4] = upper_bytes(x[0][1], x[1][1]);
          pc[i / 4] = upper_bytes(x[0][2], x[1][2]);
        }
        uint8_t *pr = sP + sb * C::PB, *prc = sPc + sb * C::PCB;
        if constexpr (R == 8) {
          *reinterpret_cast<uint4*>(pr + swz<N>(key_in, 0)) = make_uint4(pa[0], pa[1], pb[0], pb[1]);
          *reinterpret_cast<uint4*>(prc + swz<NC>(key_in, 0)) = make_uint4(0, 0, pc[0], pc[1]);
        } else if constexpr (RW == 8) {
          const int half = wg % 2 * 8;
          *reinterpret_cast<uint2*>(pr + swz<N>(key_in, wg / 2) + half) = make_uint2(pa[0], pa[1]);
          *reinterpret_cast<uint2*>(pr + swz<N>(key_in, R / 16 + wg / 2) + half) = make_uint2(pb[0], pb[1]);
          *reinterpret_cast<uint2*>(prc + swz<NC>(key_in, wg / 2) + half) = make_uint2(pc[0], pc[1]);
        } else {
          *reinterpret_cast<uint4*>(pr + swz<N>(key_in, wg)) = make_uint4(pa[0], pa[1], pa[2], pa[3]);
          *reinterpret_cast<uint4*>(pr + swz<N>(key_in, R / 16 + wg)) = make_uint4(pb[0], pb[1], pb[2], pb[3]);
          *reinterpret_cast<uint4*>(prc + swz<NC>(key_in, wg)) = make_uint4(pc[0], pc[1], pc[2], pc[3]);
        }
        if (!mine && wg == 0) {
          // a key that is not there: its value row is whatever lies in the slot, and 0·NaN is NaN
          wait_bar(&vfull[vslot], vturn, abort);
          uint8_t* v = sV + vslot * C::SLOT + key_in * CW;
#pragma unroll
          for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int k = 0; k < CW / 16; ++k) *reinterpret_cast<uint4*>(v + cb * (TILE * CW) + k * 16) = make_uint4(0, 0, 0, 0);
        }
        if (++vslot == NSV) {
          vslot = 0;
          vturn ^= 1u;
        }
        tc::fence_before();
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&pfull[sb]);
      }

      // ---- the piece is done. The scores of its last tile are here, so Q is free for the next piece, whose first
      // product then runs beside the rest: l over the keys, O out of TMEM (thread = head dim).
      if (!AHEAD && more) load_q(piece_at(piece + 1));
      if (more) stage_q(piece + 1);
      // gates, as they are in memory (whatever is done beside a load waits for it): they come in while the sums
      // are added
      uint16_t gates[CB * RW];
      if (p.whole) {
#pragma unroll
        for (int mb = 0; mb < CB; ++mb) {
          const int dim = mb * 128 + key_in;
          int h = h_first;
          const uint16_t* at = static_cast<const uint16_t*>(L.qkv) + ((int64_t)p.b * L.tokens + t_first) * L.ld_qkv +
                               (int64_t)(p.g * nrep + h) * 2 * HD + HD + dim;
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            gates[mb * RW + i] = 0;
            if (row0 + i < rows_total && dim < HD) gates[mb * RW + i] = *at;
            at += 2 * HD;
            if (++h == nrep) {
              h = 0;
              at += L.ld_qkv - (int64_t)nrep * 2 * HD;
            }
          }
        }
      }
      const float s = warp_transpose_reduce<RW, false>(l, lane);
      if (reducer) red[wg * 4 * RW + row_of<RW>(lane) * 4 + wq] = s;
      bar_sync(bar);
      if (wq == 0 && reducer) {
        const float4 v4 = *reinterpret_cast<const float4*>(red + wg * 4 * RW + row_of<RW>(lane) * 4);
        const float v = (v4.x + v4.y) + (v4.z + v4.w);
        aux[my_row] = v == 0.f ? 0.f : 1.f / v;
        if (!p.whole) ws.ml[(int64_t)p.slot * R + my_row] = make_float2(v == 0.f ? -INFINITY : mcur[my_row], v);
        mcur[my_row] = NOTHING;
      }
      wait_bar(&pdone[(tile - 1) & 1], ((tile - 1) >> 1) & 1, abort);
      tc::fence_after();
      bar_sync(bar);
#pragma unroll
      for (int mb = 0; mb < CB; ++mb) {
        const int dim = mb * 128 + key_in;
        int h = h_first;
        __nv_bfloat16* at = static_cast<__nv_bfloat16*>(L.out) + ((int64_t)p.b * L.tokens + t_first) * L.ld_out + (int64_t)(p.g * nrep + h) * HD + dim;
#pragma unroll
        for (int i0 = 0; i0 < RW; i0 += 8) {
          uint32_t oh[8], ol[8];
          tm_ld8(tout + mb * N + i0, oh);
          tm_ld8(tout + mb * N + R + i0, ol);
          tm_wait_ld8(oh, ol);
          if (p.whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float g = __uint_as_float((uint32_t)gates[mb * RW + i0 + i] << 16);
              const float v = fmaf(__uint_as_float(ol[i]), 0.25f, __uint_as_float(oh[i])) * aux[r0 + i0 + i] * sigmoid_ex2(g);
              if (row0 + i0 + i < rows_total && dim < HD) *at = __float2bfloat16_rn(v);
              at += HD;
              if (++h == nrep) {
                h = 0;
                at += L.ld_out - (int64_t)nrep * HD;
              }
            }
          } else if (dim < HD) {
            float* to = ws.o + ((int64_t)p.slot * R + r0 + i0) * HD + dim;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i * HD] = fmaf(__uint_as_float(ol[i]), 0.25f, __uint_as_float(oh[i]));
          }
          __syncwarp();
        }
      }
      tc::fence_before();   // the next piece's products overwrite O after its pfull
      ++piece;
      p = agreed_piece_at(piece);   // a barrier: aux and red are written again
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

// CTAs: one an SM, or two where registers and shared memory have room
int tc_grid(int hd, int R) { return tc::sm_count() * (hd == 256 || R >= 32 ? 1 : 2); }

// the least R that holds all query rows of a kv head, so that each key is read once; over 64 rows: units of 128, of
// rows_kernel
int tc_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

template <int HD, int R>
static int launch_tc_t(const qsp_attn_kv8_layer& L, const CUtensorMap& mk, const CUtensorMap& mv, int box_rows, cudaStream_t st) {
  using C = Cfg<HD, R>;
  auto kern = tc_kernel<HD, R>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::BYTES);
  if (e != cudaSuccess) return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: %s", cudaGetErrorString(e));
  const int n_rg = (L.n_heads / L.n_kv_heads * L.tokens + R - 1) / R, G = grid_for(L, n_rg, TILE, tc_grid(HD, R));
  const int rc = launch_pdl("qsp_attn_kv8_verify", kern, dim3(G), dim3(C::THREADS), C::BYTES, st, mk, mv, L, n_rg, box_rows);
  return rc ? rc : launch_merge(L, G, R, TILE, st);
}

template <int HD>
static int launch_tc_hd(const qsp_attn_kv8_layer& L, int R, const CUtensorMap& mk, const CUtensorMap& mv, int box_rows,
                        cudaStream_t st) {
  switch (R) {
    case 8: return launch_tc_t<HD, 8>(L, mk, mv, box_rows, st);
    case 16: return launch_tc_t<HD, 16>(L, mk, mv, box_rows, st);
    case 32: return launch_tc_t<HD, 32>(L, mk, mv, box_rows, st);
    default: return launch_tc_t<HD, 64>(L, mk, mv, box_rows, st);
  }
}

int launch_tc(const qsp_attn_kv8_layer& L, cudaStream_t st) {
  // rows of the pages are 32-bit coordinates of the tensor map
  const int64_t rows = (int64_t)L.num_pages * L.n_kv_heads * L.page_size;
  if (L.page_size % 8 != 0 || rows >= (1ll << 31)) return QSP_ERR_UNSUPPORTED;
  int box_rows = 8;
  while (box_rows < TILE && L.page_size % (2 * box_rows) == 0) box_rows *= 2;
  CUtensorMap mk, mv;
  if (!make_map(&mk, L.k_pages, rows, L.head_dim, box_rows) || !make_map(&mv, L.v_pages, rows, L.head_dim, box_rows))
    return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: no tensor map for the pages");
  const int R = tc_rows(L.n_heads / L.n_kv_heads * L.tokens);
  // rows_kernel takes the scales of 8 keys at a time; with smaller blocks: groups of 64 rows (8 x 127 tokens over 1-2k keys
  // 72 us, where it takes 52)
  if (R == 128 && L.scale_block >= GROUP) return launch_rows(L, mk, mv, box_rows, st);
  switch (L.head_dim) {
    case 32: return launch_tc_hd<32>(L, R, mk, mv, box_rows, st);
    case 64: return launch_tc_hd<64>(L, R, mk, mv, box_rows, st);
    case 128: return launch_tc_hd<128>(L, R, mk, mv, box_rows, st);
    default: return launch_tc_hd<256>(L, R, mk, mv, box_rows, st);
  }
}

int device_error(int reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv8_error, sizeof(int));
  if (reset && v) {
    const int z = 0;
    cudaMemcpyToSymbol(g_kv8_error, &z, sizeof(int));
  }
  const int rows = rows_error(reset);
  return v ? v : rows;
}

}  // namespace kv8
}  // namespace qsp
