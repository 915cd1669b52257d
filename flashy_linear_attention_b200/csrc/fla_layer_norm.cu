// Layer norm for sm_100a, with or without a residual that is added first:
//     s = x + residual (rounded to the type of the rows),   m = mean(s),   r = 1 / sqrt(mean((s - m)^2) + eps),
//     y = (s - m) r w + b,
// and with n = (s - m) r, u = dy w its gradients
//     ds' = r (u - mean(u) - n mean(u n)) + ds,   dw = sum over rows of dy n,   db = sum over rows of dy.
// The reference has no counterpart; its outputs are unnormalised (flashlinear/linear_attn.py:11-31), and a norm of the
// heads is the usual alternative to the denominator of README.md:27-30.
//
// Bound by HBM: a row is read once, into registers, and everything that is summed over it is summed from there (the
// variance from differences to the mean: no cancellation). A row has a group of 8, 16 or 32 lanes, the smallest whose
// 16-byte pieces cover it (four to a lane at most), or a CTA where it is longer. Backward, a group adds
// up its rows' dy n and dy in registers, the groups of a CTA join theirs in shared memory, and a second kernel sums the
// CTAs'. All orders are fixed.
#include <algorithm>
#include <type_traits>

#include "fla_internal.h"
#include "fla_pairs.cuh"

namespace fla {

struct NormRows {
  char* ptr;
  long long sh, s0, s1, s2;  // bytes: from head to head (weights of the heads' own), and in the three dims of the rows
};

struct LayerNormParams {
  NormRows x, z, s, y;    // forward: rows, residual (null: none), their sum (output), result
  NormRows dy, ds, dx;    // backward: x is what was normalised; ds null: none; dx null: not wanted
  const void* w;          // [heads][d] or null
  const void* b;
  int w_wide;             // weights are fp32 (else of the rows' type)
  float* stats;           // [heads][rows][2]: mean, r; null: not wanted (forward)
  float* parts;           // backward: [CTA][2][heads][d], or null
  long long rows;         // of a head
  int heads, n1, n2, d;   // row j is (j / n2 / n1, j / n2 % n1, j % n2)
  int lanes;              // that hold a piece (rows of a CTA each)
  float eps;
};

__device__ __forceinline__ long long row_offset(const NormRows& t, const LayerNormParams& p, long long j, int head) {
  if (p.n1 == 1 && p.rows == p.n2) return head * t.sh + j * t.s2;
  const unsigned row = static_cast<unsigned>(j), outer = row / static_cast<unsigned>(p.n2);  // (rows fit 31 bits)
  const unsigned i2 = row - outer * p.n2, i0 = outer / static_cast<unsigned>(p.n1), i1 = outer - i0 * p.n1;
  return head * t.sh + i0 * t.s0 + i1 * t.s1 + i2 * t.s2;
}

// A piece of a row: 16 bytes, or one element where rows are not aligned or end inside a piece.
template <typename T, bool WIDE>
struct Piece {
  static constexpr int kElements = WIDE ? 16 / sizeof(T) : 1;
  using Raw = std::conditional_t<WIDE, uint4, typename PairOf<T>::Element>;
};
template <typename T>
__device__ __forceinline__ void widen(float (&v)[16 / sizeof(T)], const uint4& raw) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(raw.x);
    v[1] = __uint_as_float(raw.y);
    v[2] = __uint_as_float(raw.z);
    v[3] = __uint_as_float(raw.w);
  } else {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_pair<T>(words[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void widen(float (&v)[1], const typename PairOf<T>::Element& raw) {
  if constexpr (sizeof(T) == 4) v[0] = raw;
  else v[0] = unpack_pair<T>(static_cast<uint32_t>(raw)).x;
}
template <typename T>
__device__ __forceinline__ void narrow(uint4& raw, const float (&v)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    raw = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    raw = make_uint4(pack_pair<T>(make_float2(v[0], v[1])), pack_pair<T>(make_float2(v[2], v[3])),
                     pack_pair<T>(make_float2(v[4], v[5])), pack_pair<T>(make_float2(v[6], v[7])));
  }
}
template <typename T>
__device__ __forceinline__ void narrow(float& raw, const float (&v)[1]) { raw = v[0]; }
template <typename T>
__device__ __forceinline__ void narrow(uint16_t& raw, const float (&v)[1]) {
  raw = static_cast<uint16_t>(pack_pair<T>(make_float2(v[0], 0.f)) & 0xffffu);
}

template <typename T, bool WIDE, int K>
struct RowRegs {
  using P = Piece<T, WIDE>;
  static constexpr int V = P::kElements;
  typename P::Raw raw[K];

  // Pieces past the row are zero.
  __device__ __forceinline__ void load(const char* row, int lane, int lanes, int d, bool in) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      raw[k] = typename P::Raw{};
      if (in && c < d) raw[k] = __ldg(reinterpret_cast<const typename P::Raw*>(row + c * static_cast<int>(sizeof(T))));
    }
  }
  __device__ __forceinline__ void store(char* row, int lane, int lanes, int d, bool in) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      if (in && c < d) *reinterpret_cast<typename P::Raw*>(row + c * static_cast<int>(sizeof(T))) = raw[k];
    }
  }
};

// A piece of the weights, of the rows' type or fp32.
template <typename T, int V>
__device__ __forceinline__ void load_weights(float (&v)[V], const void* w, int wide, long long at, bool in) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  if (!in) return;
  if (wide || sizeof(T) == 4) {
    const float* f = static_cast<const float*>(w) + at;
    if constexpr (V == 1) {
      v[0] = __ldg(f);
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(f + i));
        v[i] = q.x;
        v[i + 1] = q.y;
        v[i + 2] = q.z;
        v[i + 3] = q.w;
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    if constexpr (V == 1) widen<T>(v, __ldg(static_cast<const uint16_t*>(w) + at));
    else widen<T>(v, __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + at)));
  }
}

// Sums of N values over the lanes of a row, the same in all of them. LANES = 0: the row has the whole CTA (of up to 32
// warps); `parts` alternates between two buffers, so that one barrier a sum is enough.
template <int LANES, int N>
__device__ __forceinline__ void sum_over_row(float (&v)[N], float (*parts)[2][32], int& turn) {
  constexpr int kSpan = LANES ? LANES : 32;
#pragma unroll
  for (int o = kSpan / 2; o > 0; o /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (LANES == 0) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) parts[turn][i][warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane < warps ? parts[turn][i][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    turn ^= 1;
  }
}

constexpr int kNormGroupThreads = 256;  // of a CTA whose rows have 32 lanes or fewer

// Threads a CTA at most, for K pieces a thread (rows of a CTA each).
constexpr int norm_cta_threads(int k) { return k <= 2 ? 512 : 1024; }

template <typename T, bool WIDE, int LANES, int K>
__global__ void __launch_bounds__(LANES ? kNormGroupThreads : norm_cta_threads(K), 1) fla_layer_norm_fwd_kernel(const LayerNormParams p) {
  using Regs = RowRegs<T, WIDE, K>;
  constexpr int V = Regs::V;
  __shared__ float parts[2][2][32];
  int turn = 0;
  const int lanes = LANES ? LANES : static_cast<int>(blockDim.x), lane = threadIdx.x % lanes;
  const int groups = blockDim.x / lanes, head = blockIdx.y;
  const float over_d = 1.f / p.d;
  // (every lane of a warp, and of a CTA that shares rows, takes the same turns)
  for (long long base = static_cast<long long>(blockIdx.x) * groups; base < p.rows; base += static_cast<long long>(gridDim.x) * groups) {
    const long long j = base + threadIdx.x / lanes;
    const bool in = j < p.rows;
    Regs x;
    x.load(p.x.ptr + (in ? row_offset(p.x, p, j, head) : 0), lane, lanes, p.d, in);
    float v[K][V], sum[1] = {0.f};
    if (p.z.ptr != nullptr) {
      Regs z;
      z.load(p.z.ptr + (in ? row_offset(p.z, p, j, head) : 0), lane, lanes, p.d, in);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float a[V], b[V];
        widen<T>(a, x.raw[k]);
        widen<T>(b, z.raw[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] += b[i];
        narrow<T>(x.raw[k], a);  // what is normalised is the sum as it is stored
      }
      x.store(p.s.ptr + (in ? row_offset(p.s, p, j, head) : 0), lane, lanes, p.d, in);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      widen<T>(v[k], x.raw[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[0] += v[k][i];
    }
    sum_over_row<LANES>(sum, parts, turn);
    const float mean = sum[0] * over_d;
    float square[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] -= mean;
        if ((k * lanes + lane) * V < p.d) square[0] = fmaf(v[k][i], v[k][i], square[0]);
      }
    sum_over_row<LANES>(square, parts, turn);
    const float r = 1.f / sqrtf(square[0] * over_d + p.eps);
    if (p.stats != nullptr && lane == 0 && in)
      *reinterpret_cast<float2*>(p.stats + 2 * (head * p.rows + j)) = make_float2(mean, r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      const long long at = static_cast<long long>(head) * p.d + c;
      float w[V], b[V];
      if (p.w != nullptr) load_weights<T>(w, p.w, p.w_wide, at, c < p.d);
      if (p.b != nullptr) load_weights<T>(b, p.b, p.w_wide, at, c < p.d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float y = v[k][i] * r;
        if (p.w != nullptr) y *= w[i];
        if (p.b != nullptr) y += b[i];
        v[k][i] = y;
      }
      narrow<T>(x.raw[k], v[k]);
    }
    x.store(p.y.ptr + (in ? row_offset(p.y, p, j, head) : 0), lane, lanes, p.d, in);
  }
}

template <typename T, bool WIDE, int LANES, int K>
__global__ void __launch_bounds__(LANES ? kNormGroupThreads : norm_cta_threads(K), 1) fla_layer_norm_bwd_kernel(const LayerNormParams p) {
  using Regs = RowRegs<T, WIDE, K>;
  constexpr int V = Regs::V;
  __shared__ float parts[2][2][32];
  extern __shared__ float joined[];  // [2][d], where a CTA has several rows at a time
  int turn = 0;
  const int lanes = LANES ? LANES : static_cast<int>(blockDim.x), lane = threadIdx.x % lanes;
  const int groups = blockDim.x / lanes, head = blockIdx.y;
  const float over_d = 1.f / p.d;
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  for (long long base = static_cast<long long>(blockIdx.x) * groups; base < p.rows; base += static_cast<long long>(gridDim.x) * groups) {
    const long long j = base + threadIdx.x / lanes;
    const bool in = j < p.rows;
    Regs x, dy;
    x.load(p.x.ptr + (in ? row_offset(p.x, p, j, head) : 0), lane, lanes, p.d, in);
    dy.load(p.dy.ptr + (in ? row_offset(p.dy, p, j, head) : 0), lane, lanes, p.d, in);
    const float2 stats = in ? __ldg(reinterpret_cast<const float2*>(p.stats + 2 * (head * p.rows + j))) : make_float2(0.f, 0.f);
    float sums[2] = {0.f, 0.f};  // of u and of u n
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      float n[V], g[V], w[V];
      widen<T>(n, x.raw[k]);
      widen<T>(g, dy.raw[k]);
      if (p.w != nullptr) load_weights<T>(w, p.w, p.w_wide, static_cast<long long>(head) * p.d + c, c < p.d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[i] = (n[i] - stats.x) * stats.y;
        if (in) dw[k][i] = fmaf(g[i], n[i], dw[k][i]);
        db[k][i] += g[i];
        const float u = p.w != nullptr ? g[i] * w[i] : g[i];
        sums[0] += u;
        sums[1] = fmaf(u, n[i], sums[1]);
      }
    }
    if (p.dx.ptr == nullptr) continue;
    sum_over_row<LANES>(sums, parts, turn);
    const float mean_u = sums[0] * over_d, mean_un = sums[1] * over_d;
    Regs ds;
    if (p.ds.ptr != nullptr) ds.load(p.ds.ptr + (in ? row_offset(p.ds, p, j, head) : 0), lane, lanes, p.d, in);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      float n[V], g[V], w[V], more[V];
      widen<T>(n, x.raw[k]);
      widen<T>(g, dy.raw[k]);
      if (p.w != nullptr) load_weights<T>(w, p.w, p.w_wide, static_cast<long long>(head) * p.d + c, c < p.d);
      if (p.ds.ptr != nullptr) widen<T>(more, ds.raw[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        n[i] = (n[i] - stats.x) * stats.y;
        const float u = p.w != nullptr ? g[i] * w[i] : g[i];
        g[i] = stats.y * (u - mean_u - n[i] * mean_un);
        if (p.ds.ptr != nullptr) g[i] += more[i];
      }
      narrow<T>(x.raw[k], g);
    }
    x.store(p.dx.ptr + (in ? row_offset(p.dx, p, j, head) : 0), lane, lanes, p.d, in);
  }
  if (p.parts == nullptr) return;
  float* out = p.parts + (static_cast<long long>(blockIdx.x) * 2 * p.heads + head) * p.d;  // dw; db lies heads * d behind
  const long long db_at = static_cast<long long>(p.heads) * p.d;
  if constexpr (LANES == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = (k * lanes + lane) * V + i;
        if (c < p.d) {
          out[c] = dw[k][i];
          out[db_at + c] = db[k][i];
        }
      }
  } else {
    const int warp = threadIdx.x / 32;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int o = LANES; o < 32; o *= 2) {
          dw[k][i] += __shfl_xor_sync(0xffffffffu, dw[k][i], o);
          db[k][i] += __shfl_xor_sync(0xffffffffu, db[k][i], o);
        }
    for (int turn_of = 0; turn_of < static_cast<int>(blockDim.x) / 32; ++turn_of) {
      if (warp == turn_of && threadIdx.x % 32 < LANES) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int c = (k * lanes + lane) * V + i;
            if (c < p.d) {
              joined[c] = turn_of ? joined[c] + dw[k][i] : dw[k][i];
              joined[p.d + c] = turn_of ? joined[p.d + c] + db[k][i] : db[k][i];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < p.d; c += blockDim.x) {
      out[c] = joined[c];
      out[db_at + c] = joined[p.d + c];
    }
  }
}

// dw and db from the CTAs' sums: 32 columns a block, eight shares of the CTAs side by side, joined in order.
template <typename W>
__global__ void __launch_bounds__(256) fla_layer_norm_weights_kernel(const float* parts, int ctas, int columns, W* dw, W* db) {
  __shared__ float shares[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, share = threadIdx.x / 32;
  W* out = blockIdx.y ? db : dw;
  if (out == nullptr) return;
  float sum = 0.f;
  if (c < columns) {
    const float* at = parts + static_cast<long long>(blockIdx.y) * columns + c;
#pragma unroll 8
    for (int i = share; i < ctas; i += 8) sum += __ldg(at + static_cast<long long>(i) * 2 * columns);
  }
  shares[share][threadIdx.x % 32] = sum;
  __syncthreads();
  if (share == 0 && c < columns) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += shares[i][threadIdx.x];
    if constexpr (sizeof(W) == 4) out[c] = sum;
    else out[c] = static_cast<W>(sum);
  }
}

}  // namespace fla

namespace {

using fla::LayerNormParams;
using fla::NormRows;

constexpr int kNormMostColumns = 32768;

int norm_element(int dtype) { return dtype == FLA_DTYPE_F32 ? 4 : 2; }

struct NormPlan {
  LayerNormParams p;
  bool wide;
  int lanes, k;      // lanes: 0 where a row has a CTA
  int threads, ctas;  // ctas: of a head
};

NormRows norm_rows(const FlaTensor& t, int size, bool heads_apart) {
  NormRows r = {};
  r.ptr = static_cast<char*>(t.ptr);
  r.s0 = t.stride_b * size;
  r.s1 = heads_apart ? 0 : t.stride_h * size;
  r.s2 = t.stride_n * size;
  r.sh = heads_apart ? t.stride_h * size : 0;
  return r;
}

NormPlan norm_plan(const FlaLayerNormArgs* a, bool backward, int sm_count) {
  NormPlan plan = {};
  LayerNormParams& p = plan.p;
  const int size = norm_element(a->dtype);
  const bool apart = a->per_head != 0;
  p.x = norm_rows(a->x, size, apart);
  p.z = norm_rows(a->residual, size, apart);
  p.s = norm_rows(a->sum, size, apart);
  p.y = norm_rows(a->y, size, apart);
  p.dy = norm_rows(a->d_y, size, apart);
  p.ds = norm_rows(a->d_sum, size, apart);
  p.dx = norm_rows(a->d_x, size, apart);
  p.w = a->weight;
  p.b = a->bias;
  p.w_wide = a->w_dtype == FLA_DTYPE_F32;
  p.stats = a->stats;
  p.heads = apart ? a->heads : 1;
  p.n1 = apart ? 1 : a->heads;
  p.n2 = a->tokens;
  p.rows = static_cast<long long>(a->batch) * p.n1 * p.n2;
  p.d = a->dim;
  p.eps = a->eps;
  NormRows* const used[] = {&p.x, backward ? &p.dy : &p.y, backward ? &p.dx : &p.s, backward ? &p.ds : &p.z};
  // neighbouring dims that are one in every tensor
  long long n0 = a->batch;
  auto every = [&](auto&& holds) {
    for (NormRows* t : used)
      if (t->ptr != nullptr && !holds(*t)) return false;
    return true;
  };
  auto shift = [&] {  // the middle dim becomes the outer one
    for (NormRows* t : used) t->s1 = t->s0;
    p.n1 = static_cast<int>(n0);
    n0 = 1;
  };
  if (p.n1 == 1) shift();
  if (n0 > 1 && p.n1 * n0 < (1LL << 31) && every([&](const NormRows& t) { return t.s0 == t.s1 * p.n1; })) {
    p.n1 = static_cast<int>(n0 * p.n1);
    n0 = 1;
  }
  if (n0 == 1 && p.n2 == 1) {
    for (NormRows* t : used) t->s2 = t->s1;
    p.n2 = p.n1;
    p.n1 = 1;
  }
  if (p.n1 > 1 && every([&](const NormRows& t) { return t.s1 == t.s2 * p.n2; })) {
    p.n2 = static_cast<int>(static_cast<long long>(p.n1) * p.n2);  // (rows fit 31 bits)
    p.n1 = static_cast<int>(n0);
    for (NormRows* t : used) t->s1 = t->s0;
  }
  const int per = 16 / size;
  auto aligned = [](const void* q, int n) { return reinterpret_cast<uintptr_t>(q) % n == 0; };
  plan.wide = p.d % per == 0 && aligned(p.w, 16) && aligned(p.b, 16) && every([&](const NormRows& t) {
                return aligned(t.ptr, 16) && (p.heads == 1 || t.sh % 16 == 0) && (n0 == 1 || t.s0 % 16 == 0) &&
                       (p.n1 == 1 || t.s1 % 16 == 0) && (p.n2 == 1 || t.s2 % 16 == 0);
              });
  const int pieces = plan.wide ? p.d / per : p.d;
  if (plan.wide) {
    if (pieces <= 128) {
      plan.lanes = pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32;
      plan.k = pieces <= 32 ? 1 : pieces <= 64 ? 2 : 4;
    } else {
      plan.k = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : pieces <= 4096 ? 4 : 8;
    }
  } else if (pieces <= 512) {
    plan.lanes = 32;
    plan.k = pieces <= 32 ? 1 : pieces <= 128 ? 4 : 16;
  } else {
    plan.k = pieces <= 8192 ? 8 : 32;
  }
  plan.threads = plan.lanes ? fla::kNormGroupThreads : (pieces + plan.k * 32 - 1) / (plan.k * 32) * 32;
  const long long groups = plan.lanes ? plan.threads / plan.lanes : 1;
  // As many CTAs as are resident together; a CTA of the backward leaves a row of sums behind, so it has 8 rows or more.
  const long long most = std::max<long long>(1, static_cast<long long>(sm_count) * (2048 / plan.threads) / (backward ? 2 : 1) / p.heads);
  const long long turns = (p.rows + groups - 1) / groups;
  plan.ctas = static_cast<int>(std::min(most, backward ? (turns + 7) / 8 : turns));
  return plan;
}

size_t norm_workspace(const NormPlan& plan) { return static_cast<size_t>(plan.ctas) * 2 * plan.p.heads * plan.p.d * sizeof(float); }

template <typename T, bool WIDE, int LANES, int K>
int norm_launch(const NormPlan& plan, bool backward, cudaStream_t stream) {
  const dim3 grid(plan.ctas, plan.p.heads);
  if (backward) {
    const int shared = LANES && plan.p.parts != nullptr ? 2 * plan.p.d * static_cast<int>(sizeof(float)) : 0;
    fla::fla_layer_norm_bwd_kernel<T, WIDE, LANES, K><<<grid, plan.threads, shared, stream>>>(plan.p);
    return fla::launched(cudaSuccess, "fla_layer_norm_bwd_kernel");
  }
  fla::fla_layer_norm_fwd_kernel<T, WIDE, LANES, K><<<grid, plan.threads, 0, stream>>>(plan.p);
  return fla::launched(cudaSuccess, "fla_layer_norm_fwd_kernel");
}

template <typename T>
int norm_launch_type(const NormPlan& plan, bool backward, cudaStream_t stream) {
  if (plan.wide) {
    if (plan.lanes == 8) return norm_launch<T, true, 8, 1>(plan, backward, stream);
    if (plan.lanes == 16) return norm_launch<T, true, 16, 1>(plan, backward, stream);
    if (plan.lanes == 32 && plan.k == 1) return norm_launch<T, true, 32, 1>(plan, backward, stream);
    if (plan.lanes == 32 && plan.k == 2) return norm_launch<T, true, 32, 2>(plan, backward, stream);
    if (plan.lanes == 32) return norm_launch<T, true, 32, 4>(plan, backward, stream);
    if (plan.k == 1) return norm_launch<T, true, 0, 1>(plan, backward, stream);
    if (plan.k == 2) return norm_launch<T, true, 0, 2>(plan, backward, stream);
    if (plan.k == 4) return norm_launch<T, true, 0, 4>(plan, backward, stream);
    if constexpr (sizeof(T) == 4) return norm_launch<T, true, 0, 8>(plan, backward, stream);
    return FLA_ERR_UNSUPPORTED;
  }
  if (plan.lanes && plan.k == 1) return norm_launch<T, false, 32, 1>(plan, backward, stream);
  if (plan.lanes && plan.k == 4) return norm_launch<T, false, 32, 4>(plan, backward, stream);
  if (plan.lanes) return norm_launch<T, false, 32, 16>(plan, backward, stream);
  if (plan.k == 8) return norm_launch<T, false, 0, 8>(plan, backward, stream);
  return norm_launch<T, false, 0, 32>(plan, backward, stream);
}

int norm_dispatch(const FlaLayerNormArgs* a, const NormPlan& plan, bool backward) {
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  if (a->dtype == FLA_DTYPE_F32) return norm_launch_type<float>(plan, backward, stream);
  if (a->dtype == FLA_DTYPE_F16) return norm_launch_type<__half>(plan, backward, stream);
  return norm_launch_type<__nv_bfloat16>(plan, backward, stream);
}

int norm_check(const FlaLayerNormArgs* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->tokens <= 0 || a->dim <= 0) return FLA_ERR_INVALID;
  if (a->dtype != FLA_DTYPE_BF16 && a->dtype != FLA_DTYPE_F16 && a->dtype != FLA_DTYPE_F32) return FLA_ERR_INVALID;
  if (a->w_dtype != a->dtype && a->w_dtype != FLA_DTYPE_F32) return FLA_ERR_INVALID;
  if (a->x.ptr == nullptr || !(a->eps >= 0.f)) return FLA_ERR_INVALID;
  if (a->dim > kNormMostColumns || (a->per_head && a->heads > 65535)) return FLA_ERR_UNSUPPORTED;
  if (static_cast<long long>(a->batch) * a->heads > 0x7fffffffLL || static_cast<long long>(a->batch) * a->heads * a->tokens > 0x7fffffffLL)
    return FLA_ERR_UNSUPPORTED;
  const int size = norm_element(a->dtype), w = norm_element(a->w_dtype);
  auto off = [](const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
  for (const FlaTensor* t : {&a->x, &a->residual, &a->sum, &a->y, &a->d_y, &a->d_sum, &a->d_x})
    if (off(t->ptr, size)) return FLA_ERR_ALIGNMENT;
  if (off(a->weight, w) || off(a->bias, w) || off(a->d_weight, w) || off(a->d_bias, w) || off(a->stats, 8) || off(a->workspace, 16))
    return FLA_ERR_ALIGNMENT;
  return FLA_OK;
}

}  // namespace

extern "C" {

size_t fla_sm100_layer_norm_workspace_bytes(const FlaLayerNormArgs* a) {
  int sm_count = 0;
  if (norm_check(a) != FLA_OK || (a->d_weight == nullptr && a->d_bias == nullptr)) return 0;
  if (fla::block_device(&sm_count) != FLA_OK) sm_count = 148;
  return norm_workspace(norm_plan(a, true, sm_count));
}

int fla_sm100_layer_norm_fwd(const FlaLayerNormArgs* a) {
  int sm_count = 0;
  if (const int rc = norm_check(a)) return rc;
  if (a->y.ptr == nullptr || (a->residual.ptr == nullptr) != (a->sum.ptr == nullptr)) return FLA_ERR_INVALID;
  (void)cudaGetLastError();
  fla::g_last_launches = 0;
  if (const int rc = fla::block_device(&sm_count)) return rc;
  return norm_dispatch(a, norm_plan(a, false, sm_count), false);
}

int fla_sm100_layer_norm_bwd(const FlaLayerNormArgs* a) {
  int sm_count = 0;
  if (const int rc = norm_check(a)) return rc;
  const bool weights = a->d_weight != nullptr || a->d_bias != nullptr;
  if (a->d_y.ptr == nullptr || a->stats == nullptr || (a->d_x.ptr == nullptr && !weights)) return FLA_ERR_INVALID;
  (void)cudaGetLastError();
  fla::g_last_launches = 0;
  if (const int rc = fla::block_device(&sm_count)) return rc;
  NormPlan plan = norm_plan(a, true, sm_count);
  if (weights) {
    if (a->workspace == nullptr || a->workspace_bytes < norm_workspace(plan)) return FLA_ERR_WORKSPACE;
    plan.p.parts = static_cast<float*>(a->workspace);
  }
  if (const int rc = norm_dispatch(a, plan, true)) return rc;
  if (!weights) return FLA_OK;
  const int columns = plan.p.heads * plan.p.d;
  const dim3 grid((columns + 31) / 32, 2);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  if (a->w_dtype == FLA_DTYPE_F32)
    fla::fla_layer_norm_weights_kernel<<<grid, 256, 0, stream>>>(plan.p.parts, plan.ctas, columns, static_cast<float*>(a->d_weight),
                                                                static_cast<float*>(a->d_bias));
  else if (a->w_dtype == FLA_DTYPE_F16)
    fla::fla_layer_norm_weights_kernel<<<grid, 256, 0, stream>>>(plan.p.parts, plan.ctas, columns, static_cast<__half*>(a->d_weight),
                                                                static_cast<__half*>(a->d_bias));
  else
    fla::fla_layer_norm_weights_kernel<<<grid, 256, 0, stream>>>(plan.p.parts, plan.ctas, columns,
                                                                static_cast<__nv_bfloat16*>(a->d_weight),
                                                                static_cast<__nv_bfloat16*>(a->d_bias));
  return fla::launched(cudaSuccess, "fla_layer_norm_weights_kernel");
}

}  // extern "C"
