// The 8-bit KV cache: prep (QK-norm, partial RoPE, quantisation into the pages), the attention
// on CUDA cores (fp32 models, and shapes outside the tensor-core kernel's), the merge of divided
// units, and the C entry points.
#include "qsp_attn_kv8.cuh"
#include "qsp_tc.cuh"

#include <algorithm>

namespace qsp {
namespace kv8 {

// ------------------------------------------------------------------ prep
// Two kinds of CTA (8 warps) in one launch. The first n_kv_jobs quantise: K and V of one (sequence,
// touched block of tokens, kv head) each, a warp a token, so that the block's largest magnitudes are
// reduced and its scales and earlier codes are rewritten by one CTA, without atomics. The others norm and
// rotate q, two token rows each, a warp two or four heads at a time. A lane holds HD/32 consecutive dims
// of a row; the rotation's other half is the same element of another lane.
//
// k is normed and rotated in fp64: with 3 mantissa bits a value next to a rounding border would
// otherwise fall to either side with the order of the sum, and a cached code lives as long as its
// sequence. There are 1/8 as many k as q heads, and B200 runs fp64 at half the fp32 rate.
//
// Small calls are bound by latency: one token 3.3 us, 64 x 4 tokens 4.2 (length, then page and row, then the block's scale).
// 16 x 127 tokens of 16 + 2 x 2 heads of 256: 13.2 us for 40 MB, bound by instructions (issued in 0.7 of the
// cycles), of which the q part alone takes 9.
constexpr int PREP_WARPS = 8, PREP_ROWS = 2;

// EPL codes of a lane, EPL bytes at dst + lane·EPL
template <int EPL>
__device__ __forceinline__ void store_codes(uint8_t* dst, int lane, const float (&x)[EPL], float inv) {
  uint32_t c[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < EPL; i += 2)
    c[i / 4] |= (uint32_t)to_e4m3x2(x[i] * inv, EPL > 1 ? x[EPL > 1 ? i + 1 : 0] * inv : 0.f) << (i % 4 * 8);
  store_bytes<EPL>(dst + lane * EPL, c[0], c[1]);
}

// a lane's elements of a row, 16-byte aligned or by themselves
template <typename T, int EPL>
__device__ __forceinline__ void store_row(T* p, int lane, const float (&y)[EPL]) {
  T* dst = p + lane * EPL;
  if constexpr (sizeof(T) == 4) {
    if constexpr (EPL % 4 == 0) {
#pragma unroll
      for (int i = 0; i < EPL; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) dst[i] = dt<T>::from_f(y[i]);
    }
  } else {
    uint32_t o[EPL > 1 ? EPL / 2 : 1];
#pragma unroll
    for (int i = 0; i < EPL; i += 2) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(y[i], EPL > 1 ? y[EPL > 1 ? i + 1 : 0] : 0.f);
      o[i / 2] = *reinterpret_cast<const uint32_t*>(&v);
    }
    if constexpr (EPL == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
    else if constexpr (EPL == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    else if constexpr (EPL == 2) *reinterpret_cast<uint32_t*>(dst) = o[0];
    else *dst = dt<T>::from_f(y[0]);
  }
}

// x -> RMS-normed times 1 + w, in 64 bits
template <typename T, int EPL>
__device__ __forceinline__ void norm_row(const Row<T, EPL>& x, const Row<T, EPL>& w, float eps, double (&y)[EPL]) {
  double ss = 0;
#pragma unroll
  for (int i = 0; i < EPL; ++i) ss += (double)x[i] * (double)x[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const double inv = rsqrt(ss / (double)(32 * EPL) + (double)eps);
#pragma unroll
  for (int i = 0; i < EPL; ++i) y[i] = (double)x[i] * inv * ((double)w[i] + (double)1);
}

// the first rd dims rotated: y[d] <- y[d]·cos[d] + (d < half ? -y[d + half] : y[d - half])·sin[d]; half is a
// whole number of lanes. cs, sn: a lane's entries of the position's table row.
template <typename T, int EPL>
__device__ __forceinline__ void rotate_row(double (&y)[EPL], const Row<T, EPL>& cs, const Row<T, EPL>& sn, int rd, int lane) {
  const int lanes = rd / 2 / EPL, d = lane * EPL;
  const bool low = d < rd / 2, in = d < rd;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const double other = __shfl_sync(0xffffffffu, y[i], low ? lane + lanes : lane - lanes);
    if (in) y[i] = y[i] * (double)cs[i] + (low ? -other : other) * (double)sn[i];
  }
}

// OCC: CTAs an SM. At 4 a thread has 64 registers and the fp64 part spills: calls whose CTAs fit three an SM take 3, and
// four heads a warp in flight (64 x 4 tokens 5.2 -> 4.2 us); for more of them occupancy counts (16 x 127 13.8 us at 3, 13.1 at 4).
template <typename T, int HD, int OCC>
__global__ void __launch_bounds__(32 * PREP_WARPS, OCC)
prep_kernel(const qsp_attn_kv8_layer L, int n_kv_jobs, int most, bool vec, bool vec_w, bool vec_rope) {
  pdl_trigger();
  constexpr int EPL = HD / 32, PREP_HEADS = OCC == 3 ? 4 : 2;
  __shared__ uint32_t red[2][PREP_WARPS];
  extern __shared__ float keys[];   // [scale_block][HD] of a quantising CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nh = L.n_heads, nkv = L.n_kv_heads, rd = L.rotary_dim;
  const T* qkv = static_cast<const T*>(L.qkv);
  const bool is_q = (int)blockIdx.x >= n_kv_jobs;
  Row<T, EPL> w, cs, sn;   // weights do not change: read before the wait
  w.load(static_cast<const T*>(is_q ? L.q_norm_w : L.k_norm_w), lane, vec_w);
  pdl_wait();
  auto load_rope = [&](int pos) {
    if (lane * EPL < rd) {
      cs.load(static_cast<const T*>(L.rope_cos) + (int64_t)pos * rd, lane, vec_rope);
      sn.load(static_cast<const T*>(L.rope_sin) + (int64_t)pos * rd, lane, vec_rope);
    }
  };

  if (is_q) {
    constexpr int WPR = PREP_WARPS / PREP_ROWS;   // warps of a row
    const int64_t m = (int64_t)(blockIdx.x - n_kv_jobs) * PREP_ROWS + warp / WPR;
    if (m >= (int64_t)L.batch * L.tokens) return;
    const int b = (int)(m / L.tokens);
    const int len = L.seq_lens[b];
    // what all heads share, as they use it: the kernel is bound by instructions
    float w1[EPL];
    const int half = rd / 2 / EPL;   // lanes
    const bool low = lane < half, in = lane * EPL < rd;
#pragma unroll
    for (int i = 0; i < EPL; ++i) w1[i] = w[i] + 1.f;
    for (int h0 = warp % WPR; h0 < nh; h0 += WPR * PREP_HEADS) {
      Row<T, EPL> x[PREP_HEADS];
#pragma unroll
      for (int i = 0; i < PREP_HEADS; ++i)
        if (h0 + i * WPR < nh) x[i].load(qkv + m * L.ld_qkv + (int64_t)(h0 + i * WPR) * 2 * HD, lane, vec);
      if (h0 < WPR) {
        // a position outside the table is flagged by the quantising CTAs; its q is rotated as position 0
        const long long at = (long long)len + (m - (int64_t)b * L.tokens);
        load_rope(at >= 0 && at < L.rope_rows ? (int)at : 0);
        if (low) sn.negate();
      }
#pragma unroll
      for (int i = 0; i < PREP_HEADS; ++i) {
        if (h0 + i * WPR < nh) {
          float y[EPL], ss = 0.f;
#pragma unroll
          for (int k = 0; k < EPL; ++k) {
            y[k] = x[i][k];
            ss = fmaf(y[k], y[k], ss);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(ss * (1.f / HD) + L.eps);
#pragma unroll
          for (int k = 0; k < EPL; ++k) {
            y[k] = y[k] * inv * w1[k];
            const float other = __shfl_sync(0xffffffffu, y[k], low ? lane + half : lane - half);
            if (in) y[k] = fmaf(other, sn[k], y[k] * cs[k]);
          }
          store_row<T, EPL>(static_cast<T*>(L.q_buf) + (m * nh + h0 + i * WPR) * HD, lane, y);
        }
      }
    }
    return;
  }

  // ---- quantise one block of one head
  int job = blockIdx.x;
  const int g = job % nkv;
  job /= nkv;
  const int b = job / most, sb = L.scale_block;
  const long long base = L.seq_lens[b];
  const long long p0 = max(base, 0ll);                   // a negative length: positions below 0 are left out
  const long long blk = p0 / sb + job % most;
  const long long lo = max(p0, blk * sb);
  const long long hi = min(base + L.tokens, (blk + 1) * sb);
  const bool any = lo < hi;
  const long long lp = lo / L.page_size;
  int page = -1;
  if (any && lo < L.rope_rows && lp < L.max_pages) page = L.page_table[(int64_t)b * L.max_pages + lp];
  const int n_new = (int)(min(hi, (long long)L.rope_rows) - lo);
  Row<T, EPL> x, v;
  auto k_row = [&](int j) {
    return qkv + ((int64_t)b * L.tokens + (lo + j - base)) * L.ld_qkv + (int64_t)nh * 2 * HD + (int64_t)g * HD;
  };
  auto load_token = [&](int j) {
    x.load(k_row(j), lane, vec);
    v.load(k_row(j) + (int64_t)nkv * HD, lane, vec);
    load_rope((int)lo + j);
  };
  if (warp < n_new) load_token(warp);   // a warp's first token while the page is looked up
  const bool ok = page >= 0 && page < L.num_pages;
  if (threadIdx.x == 0 && L.bad_index != nullptr && (base < 0 || (any && (!ok || hi > L.rope_rows)))) *L.bad_index = 1;
  if (!ok) return;
  const int n_old = (int)(lo - blk * sb);
  const int slot0 = (int)(blk * sb % L.page_size);
  const int64_t ph = (int64_t)page * nkv + g;
  uint8_t* codes[2] = {static_cast<uint8_t*>(L.k_pages) + (ph * L.page_size + slot0) * HD,
                       static_cast<uint8_t*>(L.v_pages) + (ph * L.page_size + slot0) * HD};
  float* scale[2] = {L.k_scales + ph * (L.page_size / sb) + slot0 / sb, L.v_scales + ph * (L.page_size / sb) + slot0 / sb};
  int e_old[2] = {-128, -128};
  if (n_old > 0) e_old[0] = exp_of(*scale[0]), e_old[1] = exp_of(*scale[1]);

  uint32_t k_max = 0, v_max = 0;
  for (int j = warp; j < n_new; j += PREP_WARPS) {
    if (j != warp) load_token(j);
    const uint32_t v_top = __reduce_max_sync(0xffffffffu, v.top());
    double z[EPL];
    norm_row<T, EPL>(x, w, L.eps, z);
    rotate_row<T, EPL>(z, cs, sn, rd, lane);
    float y[EPL];
    uint32_t k_top = 0;
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
      y[k] = (float)z[k];
      k_top = max(k_top, __float_as_uint(y[k]) & 0x7fffffffu);
    }
    k_top = __reduce_max_sync(0xffffffffu, k_top);
    const bool fine = k_top < NOT_FINITE && v_top < NOT_FINITE;
    if (fine) k_max = max(k_max, k_top);
    if (v_top < NOT_FINITE) v_max = max(v_max, v_top);
#pragma unroll
    for (int k = 0; k < EPL; ++k) keys[j * HD + lane * EPL + k] = fine ? y[k] : NAN;
  }
  if (lane == 0) {
    red[0][warp] = k_max;
    red[1][warp] = v_max;
  }
  __syncthreads();
  int e[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t top = red[kv][0];
#pragma unroll
    for (int i = 1; i < PREP_WARPS; ++i) top = max(top, red[kv][i]);
    e[kv] = min(max(scale_exp(top), e_old[kv]), MAX_EXP);
    if (threadIdx.x == 0) *scale[kv] = exp2i(e[kv]);
    if (e_old[kv] < e[kv] && n_old > 0) {   // earlier tokens of the block take the larger scale
      const float f = ldexpf(1.f, e_old[kv] - e[kv]);
      uint32_t* c4 = reinterpret_cast<uint32_t*>(codes[kv]);
      for (int k = threadIdx.x; k < n_old * (HD / 4); k += 32 * PREP_WARPS) {
        const uint32_t c = c4[k];
        const float2 a = from_e4m3x2((uint16_t)c), z = from_e4m3x2((uint16_t)(c >> 16));
        c4[k] = (uint32_t)to_e4m3x2(a.x * f, a.y * f) | (uint32_t)to_e4m3x2(z.x * f, z.y * f) << 16;
      }
    }
  }
  for (int j = warp; j < n_new; j += PREP_WARPS) {   // a warp's own tokens again
    float y[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) y[i] = keys[j * HD + lane * EPL + i];
    store_codes<EPL>(codes[0] + (int64_t)(n_old + j) * HD, lane, y, exp2i(-e[0]));
    if (n_new > PREP_WARPS) v.load(k_row(j) + (int64_t)nkv * HD, lane, vec);
    const bool fine = __reduce_max_sync(0xffffffffu, v.top()) < NOT_FINITE;
#pragma unroll
    for (int i = 0; i < EPL; ++i) y[i] = fine ? v[i] : 0.f;
    store_codes<EPL>(codes[1] + (int64_t)(n_old + j) * HD, lane, y, exp2i(-e[1]));
  }
}

template <typename T, int HD>
static int launch_prep(const qsp_attn_kv8_layer& L, cudaStream_t st) {
  const int sb = L.scale_block;
  const int64_t most = (L.tokens + sb - 2) / sb + 1;    // blocks that T tokens can touch
  const int64_t jobs = most * L.n_kv_heads * L.batch;
  const int64_t rows = ((int64_t)L.batch * L.tokens + PREP_ROWS - 1) / PREP_ROWS;
  QSP_REQUIRE(jobs + rows < (1ll << 31), "qsp_attn_kv8_prep: too many tokens for one call");
  constexpr int A = std::min<int>(16, HD / 32 * sizeof(T));
  const bool vec = aligned(L.qkv, A) && (L.ld_qkv * (int64_t)sizeof(T)) % A == 0;
  const bool vec_w = aligned(L.q_norm_w, A) && aligned(L.k_norm_w, A);
  const bool vec_rope = aligned(L.rope_cos, A) && aligned(L.rope_sin, A) && (L.rotary_dim * (int64_t)sizeof(T)) % A == 0;
  const size_t smem = (size_t)sb * HD * sizeof(float);
  auto kern = jobs + rows <= 3 * tc::sm_count() ? prep_kernel<T, HD, 3> : prep_kernel<T, HD, 4>;
  if (smem > 40 * 1024) {   // past the 48 KB that need no leave
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_prep: %s", cudaGetErrorString(e));
  }
  return launch_pdl("qsp_attn_kv8_prep", kern, dim3((unsigned)(jobs + rows)), dim3(32 * PREP_WARPS), smem, st, L, (int)jobs,
                    (int)most, vec, vec_w, vec_rope);
}

// ------------------------------------------------------------------ attention on CUDA cores
// fp32 throughout: for fp32 models, and for bf16 shapes that the tensor-core kernel does not take.
// A CTA of 4 warps runs its pieces (see Piece) with 16 query rows, 4 a warp, and stages 32 keys at a time
// as fp32 values, the next ones' codes in flight meanwhile. Scores: lane = key, a 16-byte read of K and of
// each of the 4 queries for 16 products. Values: lane = HD/32 dims, the weights read back from shared memory.
// 3 sequences x 5 tokens over 90 to 201 keys, 8 heads of 64: 10.4 us with the merge, bound by the chain of a tile.
constexpr int SIMT_R = 16, SIMT_WARPS = 4, SIMT_RPW = SIMT_R / SIMT_WARPS;

template <typename T, int HD>
struct SimtSmem {
  float q[SIMT_R][HD];
  float k[SIMT_TILE][HD + 4];   // lanes read 16 bytes a row: the rows' banks step by 4
  float v[SIMT_TILE][HD];
  float p[SIMT_WARPS][SIMT_RPW][SIMT_TILE];
  int sh[68];
};

template <typename T, int HD>
__global__ void __launch_bounds__(32 * SIMT_WARPS) simt_kernel(const qsp_attn_kv8_layer L, int n_rg) {
  pdl_trigger();
  pdl_wait();
  constexpr int DPL = HD / 32, RPW = SIMT_RPW, THREADS = 32 * SIMT_WARPS;
  constexpr int TPK = THREADS / SIMT_TILE, CPT = HD / TPK;   // threads of a key, its codes of each
  extern __shared__ __align__(16) uint8_t simt_raw[];
  SimtSmem<T, HD>& sm = *reinterpret_cast<SimtSmem<T, HD>*>(simt_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nrep = L.n_heads / L.n_kv_heads, rows_total = nrep * L.tokens;
  const int cap = L.max_pages * L.page_size, nb = L.page_size / L.scale_block;
  const uint8_t* kp = static_cast<const uint8_t*>(L.k_pages);
  const uint8_t* vp = static_cast<const uint8_t*>(L.v_pages);
  const Scratch ws = scratch(L, gridDim.x, SIMT_R);
  const float sl2 = L.scale * LOG2E;
  const int my_key = tid / TPK, my_dim = tid % TPK * CPT;   // this thread's part of a staged tile

  Walk w = share<SIMT_TILE>(L, n_rg, SIMT_R, sm.sh);
  Piece p;
  p.n = 0;
  while (next_piece<SIMT_TILE>(L, n_rg, SIMT_R, w, p)) {
    const int row0 = p.rg * SIMT_R, nrows = min(SIMT_R, rows_total - row0);
    const int base = min(p.len, cap), kv_end = min(base + L.tokens, cap);
    // codes and scales of a tile's key; a key without a page is zeros (and not seen)
    uint32_t kc[CPT / 4], vc[CPT / 4];
    float ks, vs;
    bool mapped;
    auto fetch = [&](int j) {
      const int key = (p.j0 + j) * SIMT_TILE + my_key;
      int page = -1;
      if (j < p.n && key < kv_end) page = L.page_table[(int64_t)p.b * L.max_pages + key / L.page_size];
      mapped = page >= 0 && page < L.num_pages;
      ks = vs = 0.f;
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) kc[i] = vc[i] = 0;
      if (mapped) {
        const int slot = key % L.page_size;
        const int64_t ph = (int64_t)page * L.n_kv_heads + p.g, off = (ph * L.page_size + slot) * HD + my_dim;
        const int64_t so = ph * nb + slot / L.scale_block;
        ks = L.k_scales[so];
        vs = L.v_scales[so];
#pragma unroll
        for (int i = 0; i < CPT / 4; ++i) {
          kc[i] = reinterpret_cast<const uint32_t*>(kp + off)[i];
          vc[i] = reinterpret_cast<const uint32_t*>(vp + off)[i];
        }
      }
    };
    fetch(0);
    __syncthreads();   // the previous piece's q has been read
    for (int e = tid; e < nrows * HD; e += THREADS) {
      const int r = e / HD, d = e % HD, t = (row0 + r) / nrep, hq = p.g * nrep + (row0 + r) % nrep;
      sm.q[r][d] = dt<T>::to_f(static_cast<const T*>(L.q_buf)[(((int64_t)p.b * L.tokens + t) * L.n_heads + hq) * HD + d]);
    }
    float acc[RPW][DPL], mrow[RPW], lrow[RPW];
    int last[RPW];   // last position the row sees
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      mrow[i] = -INFINITY;
      lrow[i] = 0.f;
      last[i] = base + (row0 + warp * RPW + i) / nrep;
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[i][j] = 0.f;
    }
    for (int j = 0; j < p.n; ++j) {
      __syncthreads();   // the previous tile has been read
#pragma unroll
      for (int i = 0; i < CPT / 4; ++i) {
        const float2 k01 = from_e4m3x2((uint16_t)kc[i]), k23 = from_e4m3x2((uint16_t)(kc[i] >> 16));
        const float2 v01 = from_e4m3x2((uint16_t)vc[i]), v23 = from_e4m3x2((uint16_t)(vc[i] >> 16));
        *reinterpret_cast<float4*>(&sm.k[my_key][my_dim + 4 * i]) = make_float4(k01.x * ks, k01.y * ks, k23.x * ks, k23.y * ks);
        *reinterpret_cast<float4*>(&sm.v[my_key][my_dim + 4 * i]) = make_float4(v01.x * vs, v01.y * vs, v23.x * vs, v23.y * vs);
      }
      if (tid % TPK == 0) sm.p[0][0][my_key] = mapped ? 1.f : 0.f;   // for a moment: which keys there are
      __syncthreads();
      const bool here = sm.p[0][0][lane] != 0.f;
      if (j + 1 < p.n) fetch(j + 1);
      __syncthreads();   // p is written below
      const int key = (p.j0 + j) * SIMT_TILE + lane;
      float sc[RPW];
#pragma unroll
      for (int i = 0; i < RPW; ++i) sc[i] = 0.f;
#pragma unroll 4
      for (int d = 0; d < HD; d += 4) {
        const float4 k = *reinterpret_cast<const float4*>(&sm.k[lane][d]);
#pragma unroll
        for (int i = 0; i < RPW; ++i) {
          const float4 q = *reinterpret_cast<const float4*>(&sm.q[warp * RPW + i][d]);
          sc[i] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, sc[i]))));
        }
      }
#pragma unroll
      for (int i = 0; i < RPW; ++i) {
        const bool vis = here && key <= last[i];
        const float s = vis ? sc[i] * sl2 : -INFINITY;
        const float mnew = fmaxf(mrow[i], warp_max(s));
        const float mref = mnew == -INFINITY ? 0.f : mnew;   // nothing to see yet (a NaN score stays NaN below)
        const float alpha = exp2f(mrow[i] - mref);
        const float pr = vis ? exp2f(s - mref) : 0.f;
        lrow[i] = lrow[i] * alpha + warp_sum(pr);
        mrow[i] = mnew;
        sm.p[warp][i][lane] = pr;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[i][d] *= alpha;
      }
      __syncwarp();
#pragma unroll 2
      for (int k0 = 0; k0 < SIMT_TILE; k0 += 4) {
        float4 pr[RPW];
#pragma unroll
        for (int i = 0; i < RPW; ++i) pr[i] = *reinterpret_cast<const float4*>(&sm.p[warp][i][k0]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          Row<float, DPL> v;
          v.load(sm.v[k0 + k], lane, true);
#pragma unroll
          for (int i = 0; i < RPW; ++i) {
            const float pk = k == 0 ? pr[i].x : k == 1 ? pr[i].y : k == 2 ? pr[i].z : pr[i].w;
#pragma unroll
            for (int d = 0; d < DPL; ++d) acc[i][d] = fmaf(pk, v[d], acc[i][d]);
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = warp * RPW + i;
      if (r >= nrows) break;
      if (p.whole()) {
        const int t = (row0 + r) / nrep, hq = p.g * nrep + (row0 + r) % nrep;
        const int64_t m = (int64_t)p.b * L.tokens + t;
        const T* gate = static_cast<const T*>(L.qkv) + m * L.ld_qkv + (int64_t)hq * 2 * HD + HD + lane * DPL;
        T* o = static_cast<T*>(L.out) + m * L.ld_out + (int64_t)hq * HD + lane * DPL;
#pragma unroll
        for (int d = 0; d < DPL; ++d) {
          const float v = lrow[i] == 0.f ? 0.f : acc[i][d] / lrow[i];
          o[d] = dt<T>::from_f(v * sigmoidf_(dt<T>::to_f(gate[d])));
        }
      } else {
        const int64_t at = (int64_t)p.slot() * SIMT_R + r;
#pragma unroll
        for (int d = 0; d < DPL; ++d) ws.o[at * HD + lane * DPL + d] = acc[i][d];
        if (lane == 0) ws.ml[at] = make_float2(mrow[i], lrow[i]);
      }
    }
  }
  if (tid == 0) put_meta(ws, w, p);
}

template <typename T, int HD>
static int launch_simt(const qsp_attn_kv8_layer& L, int G, cudaStream_t st) {
  const int rows = L.n_heads / L.n_kv_heads * L.tokens, n_rg = (rows + SIMT_R - 1) / SIMT_R;
  const size_t smem = sizeof(SimtSmem<T, HD>);
  auto kern = simt_kernel<T, HD>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return set_error(QSP_ERR_CUDA, "qsp_attn_kv8_verify: %s", cudaGetErrorString(e));
  G = grid_for(L, n_rg, SIMT_TILE, G);
  const int rc = launch_pdl("qsp_attn_kv8_verify(simt)", kern, dim3(G), dim3(32 * SIMT_WARPS), smem, st, L, n_rg);
  return rc ? rc : launch_merge(L, G, SIMT_R, SIMT_TILE, st);
}

// ------------------------------------------------------------------ merge of divided units
// CTA (c, y): `each` times 8 rows, a warp each, of the divided unit whose first tile attention CTA c had, if there is one;
// or (WIDE, for few units of many parts) CTA (u, r): row r of the u-th divided unit, its partials dealt out to 8
// warps. A warp weights its partials with 2^(m_p − M) and adds them in their order, a lane HD/32 columns, four
// in flight at a time; WIDE adds the warps' sums in order. Then / l and the gate. Bound by latency: the
// launch and two dependent reads (meta; everything else).
constexpr int MERGE_WARPS = 8;

template <typename T, int HD, bool WIDE>
__global__ void __launch_bounds__(32 * MERGE_WARPS, 3) merge_kernel(const qsp_attn_kv8_layer L, int G, int R, int each, bool vec) {
  pdl_trigger();
  pdl_wait();
  constexpr int EPL = HD / 32, DEPTH = 4;
  __shared__ float part[WIDE ? MERGE_WARPS : 1][HD + 1];
  __shared__ float part_m[MERGE_WARPS];
  const Scratch ws = scratch(L, G, R);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int c = blockIdx.x;
  if constexpr (WIDE) {
    // the attention CTA that has the first tile of the u-th divided unit: thread i looks at CTAs i, i + 256, ..
    constexpr int MAX_SCAN = 4;
    __shared__ int found, counts[32];
    bool has[MAX_SCAN];
    uint32_t mask[MAX_SCAN];
#pragma unroll
    for (int k = 0; k < MAX_SCAN; ++k) {
      const int i = k * 32 * MERGE_WARPS + threadIdx.x;
      has[k] = i < G && ws.meta[i].w != 0;
    }
    if (threadIdx.x == 0) found = -1;
#pragma unroll
    for (int k = 0; k < MAX_SCAN; ++k) {
      mask[k] = __ballot_sync(0xffffffffu, has[k]);
      if (lane == 0) counts[k * MERGE_WARPS + warp] = __popc(mask[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MAX_SCAN; ++k) {
      const int w = k * MERGE_WARPS + warp;
      const int before = __reduce_add_sync(0xffffffffu, lane < w ? counts[lane] : 0);
      if (has[k] && before + __popc(mask[k] & ((1u << lane) - 1)) == (int)blockIdx.x) found = k * 32 * MERGE_WARPS + threadIdx.x;
    }
    __syncthreads();
    c = found;
    if (c < 0) return;
  }
  const int4 meta = ws.meta[c];
  const int np = meta.w, nrep = L.n_heads / L.n_kv_heads, first = 2 * c + (meta.z >> 30);
  if (np == 0) return;
#pragma unroll 1
  for (int it = 0; it < each; ++it) {
    const int r = WIDE ? blockIdx.y : (blockIdx.y * each + it) * MERGE_WARPS + warp, rr = meta.y * R + r;
    if (r >= R || rr >= nrep * L.tokens) return;   // the same for the whole CTA if WIDE
    auto slot = [&](int q) { return (int64_t)(q == 0 ? first : 2 * (c + q)) * R + r; };
    const int t = rr / nrep, hq = (meta.z & ((1 << 30) - 1)) * nrep + rr - t * nrep;
    const int64_t m = (int64_t)meta.x * L.tokens + t;
    Row<T, EPL> gate;
    gate.load(static_cast<const T*>(L.qkv) + m * L.ld_qkv + (int64_t)hq * 2 * HD + HD, lane, vec);
    float acc[EPL], den = 0.f, M = -INFINITY;   // sums relative to 2^M, the largest so far
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
    const int per = WIDE ? (np + MERGE_WARPS - 1) / MERGE_WARPS : np;
    const int q_begin = WIDE ? warp * per : 0, q_end = min(np, q_begin + per);
    for (int q0 = q_begin; q0 < q_end; q0 += DEPTH) {
      Row<float, EPL> v[DEPTH];
      float2 ml[DEPTH];
      float top = M;
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        ml[u] = make_float2(-INFINITY, 0.f);
        v[u].zero();
        if (q0 + u < q_end) {
          ml[u] = ws.ml[slot(q0 + u)];
          v[u].load(ws.o + slot(q0 + u) * HD, lane, true);
        }
      }
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) top = fmaxf(top, ml[u].x);
      const float ref = top == -INFINITY ? 0.f : top, old = exp2f(M - ref);
      M = top;
      den *= old;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] *= old;
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        if (ml[u].y != 0.f) {   // else a part of which the row saw nothing
          const float f = exp2f(ml[u].x - ref);
          den = fmaf(f, ml[u].y, den);
#pragma unroll
          for (int i = 0; i < EPL; ++i) acc[i] = fmaf(f, v[u][i], acc[i]);
        }
      }
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) part[warp][lane * EPL + i] = acc[i];
      if (lane == 0) {
        part[warp][HD] = den;
        part_m[warp] = M;
      }
      __syncthreads();
      if (warp != 0) return;
      float top = M;
#pragma unroll
      for (int w = 1; w < MERGE_WARPS; ++w) top = fmaxf(top, part_m[w]);
      const float ref = top == -INFINITY ? 0.f : top;
      den = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
#pragma unroll
      for (int w = 0; w < MERGE_WARPS; ++w) {
        const float f = exp2f(part_m[w] - ref);
        den = fmaf(f, part[w][HD], den);
#pragma unroll
        for (int i = 0; i < EPL; ++i) acc[i] = fmaf(f, part[w][lane * EPL + i], acc[i]);
      }
    }
    T* out = static_cast<T*>(L.out) + m * L.ld_out + (int64_t)hq * HD;
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = acc[i] * inv * sigmoidf_(gate[i]);
    if (vec) {
      store_row<T, EPL>(out, lane, acc);
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) out[lane * EPL + i] = dt<T>::from_f(acc[i]);
    }
  }
}

template <typename T, int HD>
static int launch_merge_hd(const qsp_attn_kv8_layer& L, int G, int R, cudaStream_t st) {
  const int rows = L.n_heads / L.n_kv_heads * L.tokens;
  const int64_t units = (int64_t)L.batch * L.n_kv_heads * ((rows + R - 1) / R);
  // few units of many parts each, and few rows: a CTA a row (one sequence of 32k keys, hd 256: 74 parts). Many rows fill the
  // GPU by themselves.
  constexpr int A = std::min<int>(16, HD / 32 * sizeof(T));
  const bool vec = aligned(L.qkv, A) && aligned(L.out, A) && (L.ld_qkv * (int64_t)sizeof(T)) % A == 0 && (L.ld_out * (int64_t)sizeof(T)) % A == 0;
  if (units * MERGE_WARPS <= G && units * std::min(R, rows) <= 2 * tc::sm_count())
    return launch_pdl("qsp_attn_kv8_verify(merge)", merge_kernel<T, HD, true>, dim3((unsigned)units, std::min(R, rows)),
                      dim3(32 * MERGE_WARPS), 0, st, L, G, R, 1, vec);
  // 128 rows of many units: fewer CTAs, most of which find nothing to do (8 x 127 tokens over 1-2k keys, all whole: 54.5 us
  // with 1, 52.5 with 4); of few units: one row a warp (1 x 128 over 16k: 60 and 70)
  const int each = R > 64 && 2 * units >= G ? 4 : 1;
  return launch_pdl("qsp_attn_kv8_verify(merge)", merge_kernel<T, HD, false>,
                    dim3(G, (std::min(R, rows) + each * MERGE_WARPS - 1) / (each * MERGE_WARPS)), dim3(32 * MERGE_WARPS), 0, st, L, G, R, each, vec);
}

template <typename T>
static int launch_merge_t(const qsp_attn_kv8_layer& L, int G, int R, cudaStream_t st) {
  switch (L.head_dim) {
    case 32: return launch_merge_hd<T, 32>(L, G, R, st);
    case 64: return launch_merge_hd<T, 64>(L, G, R, st);
    case 128: return launch_merge_hd<T, 128>(L, G, R, st);
    default: return launch_merge_hd<T, 256>(L, G, R, st);
  }
}

int launch_merge(const qsp_attn_kv8_layer& L, int G, int R, int keys, cudaStream_t st) {
  // none is divided where units have one tile, or where share() cannot but leave all whole: as many CTAs as units, none
  // of more than merge_cost (16 x 17 tokens over 700 keys: 30.6 us with the launch, 26.8 without)
  const int64_t tiles = ((int64_t)L.max_pages * L.page_size + keys - 1) / keys;
  const int64_t units = (int64_t)L.batch * L.n_kv_heads * ((L.n_heads / L.n_kv_heads * L.tokens + R - 1) / R);
  if (tiles <= 1 || (units <= G && UNIT_COST + tiles <= merge_cost(R))) return QSP_OK;
  QSP_DISPATCH_DTYPE(L.dtype, T, { return launch_merge_t<T>(L, G, R, st); });
}

// CTAs of the CUDA-core kernel: two fit an SM at head_dim 256 (83 KB of shared memory each)
static int simt_grid() { return 2 * tc::sm_count(); }

static int validate(const char* what, const qsp_attn_kv8_layer* p, bool verify) {
  QSP_REQUIRE(p != nullptr, "%s: null layer", what);
  const qsp_attn_kv8_layer& L = *p;
  QSP_REQUIRE(L.qkv && L.k_pages && L.v_pages && L.k_scales && L.v_scales && L.page_table && L.seq_lens && L.q_buf,
              "%s: null pointer", what);
  QSP_REQUIRE(L.batch > 0 && L.tokens > 0 && (int64_t)L.batch * L.tokens < (1 << 30), "%s: bad batch/tokens", what);
  QSP_REQUIRE(L.n_heads > 0 && L.n_kv_heads > 0 && L.n_heads % L.n_kv_heads == 0 && L.n_heads <= (1 << 16),
              "%s: n_heads must be a multiple of n_kv_heads", what);
  QSP_REQUIRE(L.head_dim == 32 || L.head_dim == 64 || L.head_dim == 128 || L.head_dim == 256, "%s: head_dim %d not built", what,
              L.head_dim);
  QSP_REQUIRE(L.page_size > 0 && L.max_pages > 0 && L.num_pages > 0 && (int64_t)L.max_pages * L.page_size < (1ll << 30),
              "%s: bad paging", what);
  QSP_REQUIRE(L.scale_block > 0 && L.scale_block <= 64 && (L.scale_block & (L.scale_block - 1)) == 0 &&
                  L.page_size % L.scale_block == 0,
              "%s: scale_block %d must be a power of two up to 64 that divides the page size %d", what, L.scale_block, L.page_size);
  const int64_t q_rows = (int64_t)L.n_heads / L.n_kv_heads * L.tokens;
  QSP_REQUIRE((double)L.batch * L.n_kv_heads * (q_rows / 8 + 1) * ((int64_t)L.max_pages * L.page_size / kv8::SIMT_TILE + 4) < 2e9,
              "%s: more than 2^31 tiles of keys", what);
  QSP_REQUIRE(aligned(L.k_pages, 16) && aligned(L.v_pages, 16) && aligned(L.q_buf, 16), "%s: pages and q_buf must be 16-byte aligned",
              what);
  QSP_REQUIRE(L.ld_qkv >= (2ll * L.n_heads + 2ll * L.n_kv_heads) * L.head_dim, "%s: ld_qkv too small", what);
  QSP_REQUIRE(L.dtype == QSP_F32 || L.dtype == QSP_BF16, "%s: unsupported dtype %d", what, L.dtype);
  if (!verify) {
    QSP_REQUIRE(L.q_norm_w && L.k_norm_w && (L.rotary_dim == 0 || (L.rope_cos && L.rope_sin)) && L.rope_rows > 0,
                "%s: null pointer or empty RoPE table", what);
    QSP_REQUIRE(L.rotary_dim >= 0 && L.rotary_dim <= L.head_dim && L.rotary_dim % (L.head_dim / 16) == 0,
                "%s: rotary_dim %d must be a multiple of head_dim / 16, head_dim at most", what, L.rotary_dim);
    return QSP_OK;
  }
  const size_t need = qsp_attn_kv8_workspace_bytes(L.batch, L.tokens, L.n_heads, L.n_kv_heads, L.head_dim, L.dtype);
  QSP_REQUIRE(L.out && L.ld_out >= (int64_t)L.n_heads * L.head_dim, "%s: missing output or ld_out too small", what);
  QSP_REQUIRE(L.workspace && aligned(L.workspace, 16) && L.workspace_bytes >= need,
              "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", what, need, L.workspace ? L.workspace_bytes : 0);
  return QSP_OK;
}

}  // namespace kv8
}  // namespace qsp

using namespace qsp;

extern "C" {

int qsp_attn_kv8_prep(const qsp_attn_kv8_layer* layer, void* stream) {
  const int rc = kv8::validate("qsp_attn_kv8_prep", layer, false);
  if (rc) return rc;
  const cudaStream_t st = as_stream(stream);
  QSP_DISPATCH_DTYPE(layer->dtype, T, {
    switch (layer->head_dim) {
      case 32: return kv8::launch_prep<T, 32>(*layer, st);
      case 64: return kv8::launch_prep<T, 64>(*layer, st);
      case 128: return kv8::launch_prep<T, 128>(*layer, st);
      default: return kv8::launch_prep<T, 256>(*layer, st);
    }
  });
}

int qsp_attn_kv8_verify(const qsp_attn_kv8_layer* layer, void* stream) {
  const int rc = kv8::validate("qsp_attn_kv8_verify", layer, true);
  if (rc) return rc;
  const cudaStream_t st = as_stream(stream);
  if (layer->dtype == QSP_BF16) {
    const int rc2 = kv8::launch_tc(*layer, st);
    if (rc2 != QSP_ERR_UNSUPPORTED) return rc2;
  }
  const int G = kv8::simt_grid();
  QSP_DISPATCH_DTYPE(layer->dtype, T, {
    switch (layer->head_dim) {
      case 32: return kv8::launch_simt<T, 32>(*layer, G, st);
      case 64: return kv8::launch_simt<T, 64>(*layer, G, st);
      case 128: return kv8::launch_simt<T, 128>(*layer, G, st);
      default: return kv8::launch_simt<T, 256>(*layer, G, st);
    }
  });
}

size_t qsp_attn_kv8_workspace_bytes(int32_t batch, int32_t tokens, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int dtype) {
  if (batch <= 0 || tokens <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 ||
      (dtype != QSP_F32 && dtype != QSP_BF16))
    return 0;
  const size_t simt = kv8::scratch_bytes(kv8::simt_grid(), kv8::SIMT_R, head_dim);
  if (dtype == QSP_F32) return simt;
  const int R = kv8::tc_rows(n_heads / n_kv_heads * std::min(tokens, 128));
  return std::max(simt, kv8::scratch_bytes(kv8::tc_grid(head_dim, R), R, head_dim));
}

}  // extern "C"
