// Shared by the kernels of the 8-bit KV cache: e4m3 conversions, power-of-two scales, and the
// division of the attention's work over the CTAs.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "qsp_common.cuh"

namespace qsp {
namespace kv8 {

constexpr int TILE = 128;      // keys of a tensor-core work tile
constexpr int SIMT_TILE = 32;  // ... of one of the CUDA-core kernel
constexpr int GROUP = 8;       // keys that share their scales in rows_kernel: scale_block is a multiple
constexpr int MIN_EXP = -40;   // least exponent of a scale
constexpr int MAX_EXP = 120;   // 448·2^120 holds every fp32 value
constexpr float LOG2E = 1.4426950408889634f;

// ---------------------------------------------------------------- e4m3
// two fp32 -> two codes (round to nearest even, saturating; NaN -> 0x7f), lo in the low byte
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return *reinterpret_cast<__half2*>(&r);
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t v) { return __half22float2(e4m3x2_to_half2(v)); }

// ---------------------------------------------------------------- a lane's elements of a row
// EPL elements at p + lane·EPL, kept as they are in memory (bf16: pairs, the low half first, each the upper
// half of an fp32)
template <typename T, int EPL>
struct Row {
  static constexpr int W = EPL * (int)sizeof(T) >= 4 ? EPL * (int)sizeof(T) / 4 : 1;
  uint32_t r[W];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r[i]);
    return __uint_as_float(i & 1 ? r[i / 2] & 0xffff0000u : r[i / 2] << 16);
  }
  // vec: the address is a multiple of min(16 bytes, EPL elements)
  __device__ __forceinline__ void load(const T* p, int lane, bool vec) {
    const T* src = p + lane * EPL;
    if (vec && W > 1) {
      if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const uint4 u = reinterpret_cast<const uint4*>(src)[i / 4];
          r[i] = u.x, r[i + 1] = u.y, r[i + 2] = u.z, r[i + 3] = u.w;
        }
      } else if constexpr (W == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(src);
        r[0] = u.x, r[1] = u.y;
      }
      return;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) r[i] = __float_as_uint(src[i]);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int i = 0; i < W; ++i) r[i] = h[2 * i] | (EPL > 1 ? (uint32_t)h[EPL > 1 ? 2 * i + 1 : 0] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = 0;
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
  }
  // bits of the largest magnitude (they compare as the values do; 0x7f800000 and over: not finite)
  __device__ __forceinline__ uint32_t top() const {
    uint32_t t = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < W; ++i) t = max(t, r[i] & 0x7fffffffu);
      return t;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) t = __vmaxu2(t, r[i] & 0x7fff7fffu);   // two halves at a time
      return max(t & 0xffff0000u, t << 16);
    }
  }
};
constexpr uint32_t NOT_FINITE = 0x7f800000u;

// N = 1, 2, 4 or 8 bytes, a first
template <int N>
__device__ __forceinline__ void store_bytes(uint8_t* dst, uint32_t a, uint32_t b) {
  if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(a, b);
  else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(dst) = a;
  else if constexpr (N == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)a;
  else *dst = (uint8_t)a;
}

// ---------------------------------------------------------------- scales
// least e in [MIN_EXP, MAX_EXP] with amax <= 448·2^e, amax finite and >= 0 given by its bits:
// 448 = 1.75·2^8, so e is amax's exponent - 8, and one more where its mantissa is over 1.75
__device__ __forceinline__ int scale_exp(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - (127 + 8) + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, MIN_EXP), MAX_EXP);
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exp_of(float scale) { return ((__float_as_int(scale) >> 23) & 0xff) - 127; }

// ---------------------------------------------------------------- work division
// A unit is (sequence b, row group rg, kv head g): `R` query rows (t, q head of the group) against
// the keys the last of them sees, cut into tiles of TILE keys. The tiles of all units, in the
// order b, rg, g, are divided evenly over the CTAs, so a ragged batch, one long sequence and many
// short ones all keep every SM equally busy. Beginning a unit counts as UNIT_COST tiles (queries in,
// output out). A CTA's share is a run of pieces (parts of units). A piece that is a whole unit is
// written out by its CTA; the others leave a partial (o, m, l) in the workspace: slot 2c for the
// first piece of CTA c, 2c + 1 for its last. The CTA that has the first tile of a divided unit
// describes it in meta[c] for the merge kernel.
// Dividing has a price: a second piece for most CTAs and the merge. Where no CTA would have more than
// merge_cost tiles less to do for it, each unit goes whole to one CTA: 64 sequences of 2048 to 2560 keys,
// 2 kv heads: 128 CTAs with at most 20 tiles each instead of 148 with 15.6 on average (37.1 us divided, 34.9 whole).
// Units of 128 rows leave partials of 128 KB (hd 256), so dividing costs more: 2 x 512 tokens over 8k keys took
// 173 us with a bound of 10 tiles, which divides them, 152 us with 12.
constexpr int UNIT_COST = 3;
__host__ __device__ __forceinline__ int merge_cost(int R) { return R > 64 ? 12 : 6; }

struct Piece {
  int b, rg, g;
  int len;          // cached tokens of the sequence
  int j0, n;        // first tile and tiles of this piece
  int unit_tiles;   // tiles of the unit
  bool first;       // the CTA's first piece
  __device__ __forceinline__ bool whole() const { return n == unit_tiles; }
  __device__ __forceinline__ int slot() const { return 2 * (int)blockIdx.x + (first ? 0 : 1); }
};

template <int KEYS>
__device__ __forceinline__ int unit_tiles(const qsp_attn_kv8_layer& L, int len, int rg, int n_rg, int R) {
  const int t_last = rg == n_rg - 1 ? L.tokens - 1 : ((rg + 1) * R - 1) / (L.n_heads / L.n_kv_heads);
  const int cap = L.max_pages * L.page_size;
  const int kv = min(min(len, cap) + t_last + 1, cap);
  return kv <= KEYS ? 1 : (kv + KEYS - 1) / KEYS;   // a unit without keys has a tile too: it writes zeros
}

// Positions count UNIT_COST + tiles for each unit; the host has checked that all fit 31 bits.
struct Walk {
  int b, rg, g;       // unit to go on at
  int at;             // position in that unit
  int pos, end;       // the same position among all, and the end of this CTA's share
  int total, parts;   // of all units, and the CTAs that share them
  int len, next_len;  // cached tokens of sequence b and (loaded ahead) of b + 1
  bool first;
};
__device__ __forceinline__ int share_begin(int c, int total, int parts) {
  const int q = total / parts, r = total - q * parts;
  return c * q + min(c, r);
}
__device__ __forceinline__ int share_owner(int pos, int total, int parts) {
  const int q = total / parts, r = total - q * parts;
  return pos < r * (q + 1) ? pos / (q + 1) : r + (pos - r * (q + 1)) / q;
}

// This CTA's share, found by all threads of the CTA; `sh` holds 68 ints of shared memory. Ends with
// a __syncthreads.
template <int KEYS>
__device__ __forceinline__ Walk share(const qsp_attn_kv8_layer& L, int n_rg, int R, int* sh) {
  const int n = L.batch * n_rg, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int per = (n + blockDim.x - 1) / blockDim.x;   // (b, rg) pairs of a thread: consecutive ones
  auto cost = [&](int i) {
    const int b = n_rg == 1 ? i : i / n_rg;
    return UNIT_COST + unit_tiles<KEYS>(L, L.seq_lens[b], i - b * n_rg, n_rg, R);
  };
  int mine = 0, most = 0;
#pragma unroll 1
  for (int k = 0; k < per; ++k) {
    if (tid * per + k < n) {
      const int one = cost(tid * per + k);
      mine += one;
      most = max(most, one);
    }
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) {
    sh[warp] = incl;
    sh[36 + warp] = most;
  }
  __syncthreads();
  const int of_warp = lane < nw ? sh[lane] : 0;
  most = __reduce_max_sync(0xffffffffu, lane < nw ? sh[36 + lane] : 0);
  const int total = __reduce_add_sync(0xffffffffu, of_warp) * L.n_kv_heads;
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0) + incl - mine;
  Walk w;
  w.total = total;
  w.first = true;
  const int units = n * L.n_kv_heads;
  if (units <= (int)gridDim.x && most <= total / (int)gridDim.x + merge_cost(R)) {
    // unit c to CTA c
    const bool any = (int)blockIdx.x < units;
    const int i = any ? blockIdx.x / L.n_kv_heads : 0;
    w.b = i / n_rg;
    w.rg = i - w.b * n_rg;
    w.g = blockIdx.x - i * L.n_kv_heads;
    w.at = w.pos = 0;
    w.len = L.seq_lens[w.b];
    w.next_len = 0;
    w.end = any ? UNIT_COST + unit_tiles<KEYS>(L, w.len, w.rg, n_rg, R) : 0;
    w.parts = 0;
    __syncthreads();
    return w;
  }
  const int parts = min((int)gridDim.x, total);   // no more CTAs than tiles: every one of them has some
  const int c = min((int)blockIdx.x, parts);
  const int begin = share_begin(c, total, parts), end = share_begin(min(c + 1, parts), total, parts);
  int a = before * L.n_kv_heads;
  if (a <= begin && begin < a + mine * L.n_kv_heads) {   // one thread's
#pragma unroll 1
    for (int k = 0; k < per; ++k) {
      const int one = cost(tid * per + k), all = one * L.n_kv_heads;
      if (begin < a + all) {
        sh[32] = tid * per + k;
        sh[33] = (begin - a) / one;
        sh[34] = (begin - a) % one;
        sh[35] = L.seq_lens[sh[32] / n_rg];
        break;
      }
      a += all;
    }
  }
  __syncthreads();
  w.b = sh[32] / n_rg;
  w.rg = sh[32] - w.b * n_rg;
  w.g = sh[33];
  w.at = sh[34];
  w.pos = begin;
  w.end = end;
  w.parts = parts;
  w.len = sh[35];
  w.next_len = begin < end && w.b + 1 < L.batch ? L.seq_lens[w.b + 1] : 0;
  return w;
}

template <int KEYS>
__device__ __forceinline__ bool next_piece(const qsp_attn_kv8_layer& L, int n_rg, int R, Walk& w, Piece& p) {
  while (w.pos < w.end) {
    p.b = w.b;
    p.rg = w.rg;
    p.g = w.g;
    p.len = w.len;
    p.unit_tiles = unit_tiles<KEYS>(L, w.len, w.rg, n_rg, R);
    const int step = min(UNIT_COST + p.unit_tiles - w.at, w.end - w.pos);
    p.j0 = max(w.at - UNIT_COST, 0);
    p.n = max(w.at + step - UNIT_COST, 0) - p.j0;
    w.pos += step;
    w.at = 0;
    if (++w.g == L.n_kv_heads) {
      w.g = 0;
      if (++w.rg == n_rg) {
        w.rg = 0;
        ++w.b;
        w.len = w.next_len;
        w.next_len = w.b + 1 < L.batch ? L.seq_lens[w.b + 1] : 0;
      }
    }
    if (p.n > 0) {
      p.first = w.first;
      w.first = false;
      return true;
    }
  }
  return false;
}

// workspace: meta [G] int4, then partials: ml [2G][R] float2 (m in log2 units, l), o [2G][R][hd]
struct Scratch {
  int4* meta;
  float2* ml;
  float* o;
};
__host__ __device__ __forceinline__ Scratch scratch(const qsp_attn_kv8_layer& L, int G, int R) {
  Scratch s;
  s.meta = static_cast<int4*>(L.workspace);
  s.ml = reinterpret_cast<float2*>(s.meta + G);
  s.o = reinterpret_cast<float*>(s.ml + 2ll * G * R);
  return s;
}
inline size_t scratch_bytes(int G, int R, int hd) { return (size_t)G * 16 + 2ull * G * R * (8 + 4ull * hd); }

// meta of this CTA: {b, rg, g | 2^30 when its partial is in slot 2c + 1, partials (0: no unit that is
// divided begins here)}. Called by one thread after the last piece `p` (p.n == 0: no piece at all).
__device__ __forceinline__ void put_meta(const Scratch& s, const Walk& w, const Piece& p) {
  int4 m = make_int4(0, 0, 0, 0);
  if (p.n > 0 && !p.whole() && p.j0 == 0) {
    const int last = w.end - p.n + p.unit_tiles - 1;   // position of the unit's last tile
    m = make_int4(p.b, p.rg, p.g | (p.first ? 0 : 1 << 30), share_owner(last, w.total, w.parts) - (int)blockIdx.x + 1);
  }
  s.meta[blockIdx.x] = m;
}

// CTAs of a launch: `most`, or as many as there can be positions
inline int grid_for(const qsp_attn_kv8_layer& L, int n_rg, int keys, int most) {
  const int64_t unit = UNIT_COST + ((int64_t)L.max_pages * L.page_size + keys - 1) / keys;
  const int64_t all = (int64_t)L.batch * L.n_kv_heads * n_rg * unit;
  return (int)(all < most ? all : most);
}
// keys: of a work tile
int launch_merge(const qsp_attn_kv8_layer& L, int G, int R, int keys, cudaStream_t st);
// the tensor-core kernels; QSP_ERR_UNSUPPORTED when the shape is not one they take
int launch_tc(const qsp_attn_kv8_layer& L, cudaStream_t st);
int tc_rows(int rows);            // their query rows per unit, for this many rows of a kv head
int tc_grid(int hd, int R);       // their CTAs
// ... for units of 128 rows; the tensor maps of K and V, boxes of box_rows keys
int launch_rows(const qsp_attn_kv8_layer& L, const CUtensorMap& mk, const CUtensorMap& mv, int box_rows, cudaStream_t st);
int device_error(int reset);
int rows_error(int reset);

}  // namespace kv8
}  // namespace qsp
