// Layer norm for sm_100a, with or without a residual that is added first:
//     s = x + residual (rounded to the type of the rows),   m = mean(s),   r = 1 / sqrt(mean((s - m)^2) + eps),
//     y = (s - m) r w + b,
// and with n = (s - m) r, u = dy w its gradients
//     ds' = r (u - mean(u) - n mean(u n)) + ds,   dw = sum over rows of dy n,   db = sum over rows of dy.
// The reference has no counterpart; its outputs are unnormalised (flashlinear/linear_attn.py:11-31), and a norm of the
// heads is the usual alternative to the denominator of README.md:27-30.
//
// Bound by HBM: a row is read once, and everything that is summed over it is summed from registers (the variance from
// differences to the mean: no cancellation). A row has a group of 4 to 32 lanes, or whole warps where it is longer; a thread
// holds 16 of its elements, which shares the shuffles, barriers and addresses of a row among more of them than 8 did
// (32768 rows of 4096 in bf16, forward: 140 us with 8, 97 with 16). Rows are on their way in shared memory
// while the ones before are worked on. Backward, a group adds up its rows' dy n and dy in registers, the groups of a CTA join
// theirs in shared memory, and a second kernel sums the CTAs'. All orders are fixed.
//
// Measured (B200, of the 6.45 TB/s of a copy), bf16: 32768 rows of 4096 forward 97 us (86 %), backward 149 (84 %), with a
// residual 194 (86 %) and 173 (96 %); 1048576 rows of 128 101 (83 %) and 150 (83 %); 524288 rows of 64 in fp16 26 us
// (79 %). Rows that are no multiple of 16 bytes go element by element: 142848 rows of 83 in fp32 33 (45 %) and 51 (43 %).
#include <algorithm>
#include <type_traits>

#include "fla_internal.h"
#include "fla_pairs.cuh"

namespace fla {

struct NormRows {
  char* ptr;
  long long sh, s0, s1, s2;  // bytes: from head to head (weights of the heads' own), and in the three dims of the rows
};

// Exact division of numbers below 2^31 by one that the host knows: with l = ceil(log2 d) and mul = floor(2^(31 + l) / d) + 1,
// mul d is above 2^(31 + l) by 2^l at most, so j mul / 2^(31 + l) is above j / d by less than 1 / d.
struct Divisor {
  unsigned d, mul, shift;
};
__device__ __forceinline__ unsigned over(unsigned j, const Divisor& d) {
  return static_cast<unsigned>(static_cast<unsigned long long>(j) * d.mul >> d.shift);
}

struct LayerNormParams {
  NormRows x, z, s, y;    // forward: rows, residual (null: none), their sum (output), result
  NormRows dy, ds, dx;    // backward: x is what was normalised; ds null: none; dx null: not wanted
  const void* w;          // [heads][d] or null
  const void* b;
  int w_wide;             // weights are fp32 (else of the rows' type)
  float* stats;           // [heads][rows][2]: mean, r, rows in the order of their indices; null: not wanted (forward)
  float* parts;           // backward: [CTA][2][heads][d], or null
  long long rows;         // of a head
  int heads, n1, n2, d;   // row j is (j / n2 / n1, j / n2 % n1, j % n2)
  Divisor by_n1, by_n2;
  Divisor stat_n1, stat_n2;  // not FLAT: row j has its statistics at the place that its indices have with these steps
  unsigned stat_step[3];
  int lanes;              // threads that share a row, where they are whole warps
  float eps;
};

// The rows that a group of threads works on, one after the other: their numbers are `step` apart. FLAT: all rows of a head
// are one stride apart in every tensor, in the order of their indices, and addresses are advanced, not worked out (64-bit products and a division for
// each row and tensor were a third of the instructions).
template <bool FLAT>
struct Cursor {
  char* at;         // FLAT: the row's address
  const NormRows* t;
  long long step_bytes;
  long long of_head;

  __device__ __forceinline__ Cursor(const NormRows& rows, int head, unsigned row, unsigned step) {
    t = &rows;
    of_head = head * rows.sh;
    if (FLAT) {
      at = rows.ptr + of_head + row * rows.s2;
      step_bytes = step * rows.s2;
    }
  }
  // Row `row`, which has to be the one that the cursor has been advanced to.
  __device__ __forceinline__ char* get(const LayerNormParams& p, unsigned row, bool in) const {
    if (FLAT) return at;
    if (!in) return t->ptr;
    const unsigned outer = over(row, p.by_n2), i2 = row - outer * p.n2;
    const unsigned i0 = over(outer, p.by_n1), i1 = outer - i0 * p.n1;
    return t->ptr + (of_head + i0 * t->s0 + i1 * t->s1 + i2 * t->s2);
  }
  __device__ __forceinline__ void advance() {
    if (FLAT) at += step_bytes;
  }
};

// Where the statistics of row j are. They go by the rows' indices and not by where these lie, since a tensor that is kept
// for the backward can come back with other strides.
template <bool FLAT>
__device__ __forceinline__ float* stats_of(const LayerNormParams& p, int head, unsigned j) {
  if (!FLAT) {
    const unsigned outer = over(j, p.stat_n2), i0 = over(outer, p.stat_n1);
    j = i0 * p.stat_step[0] + (outer - i0 * p.stat_n1.d) * p.stat_step[1] + (j - outer * p.stat_n2.d) * p.stat_step[2];
  }
  return p.stats + 2 * (head * p.rows + j);
}

// A piece of a row: 16 bytes, or one element where rows are not aligned or end inside a piece.
template <typename T, bool WIDE>
struct Piece {
  static constexpr int kElements = WIDE ? 16 / sizeof(T) : 1;
  using Raw = std::conditional_t<WIDE, uint4, typename PairOf<T>::Element>;
};

// Loads where `ok`, and leaves the register as it is elsewhere. As one predicated instruction: as a branch or a selection
// the compiler waited for the loads of later rows before it went on.
__device__ __forceinline__ void load_if(uint4& r, const char* p, bool ok) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %5, 0;\n\t@p ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
               : "l"(p), "r"(static_cast<int>(ok)));
}
__device__ __forceinline__ void load_if(float& r, const char* p, bool ok) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p ld.global.nc.f32 %0, [%1];\n\t}"
               : "+f"(r)
               : "l"(p), "r"(static_cast<int>(ok)));
}
__device__ __forceinline__ void load_if(uint16_t& r, const char* p, bool ok) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p ld.global.nc.b16 %0, [%1];\n\t}"
               : "+h"(r)
               : "l"(p), "r"(static_cast<int>(ok)));
}

// What a thread holds of a row: K pieces, in memory `lanes` pieces apart. In arithmetic the elements go in pairs.
template <typename T, bool WIDE, int K>
struct RowRegs {
  using Raw = typename Piece<T, WIDE>::Raw;
  static constexpr int V = Piece<T, WIDE>::kElements, kPairs = K * V / 2;
  Raw raw[K];

  // Pieces past the row are zero.
  __device__ __forceinline__ void load(const char* row, int lane, int lanes, int d, bool in) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      raw[k] = Raw{};
      load_if(raw[k], row + c * static_cast<int>(sizeof(T)), in && c < d);
    }
  }
  __device__ __forceinline__ void store(char* row, int lane, int lanes, int d, bool in) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * lanes + lane) * V;
      if (in && c < d) *reinterpret_cast<Raw*>(row + c * static_cast<int>(sizeof(T))) = raw[k];
    }
  }
  __device__ __forceinline__ void widen(float2 (&v)[kPairs]) const {
    if constexpr (!WIDE) {
#pragma unroll
      for (int k = 0; k < K; k += 2) v[k / 2] = unpack_pair<T>(join_pair(raw[k], raw[k + 1]));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[2 * k] = make_float2(__uint_as_float(raw[k].x), __uint_as_float(raw[k].y));
        v[2 * k + 1] = make_float2(__uint_as_float(raw[k].z), __uint_as_float(raw[k].w));
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[4 * k] = unpack_pair<T>(raw[k].x);
        v[4 * k + 1] = unpack_pair<T>(raw[k].y);
        v[4 * k + 2] = unpack_pair<T>(raw[k].z);
        v[4 * k + 3] = unpack_pair<T>(raw[k].w);
      }
    }
  }
  // Rounded to nearest, once.
  __device__ __forceinline__ void narrow(const float2 (&v)[kPairs]) {
    if constexpr (!WIDE) {
#pragma unroll
      for (int k = 0; k < K; k += 2) {
        const auto r = pack_pair<T>(v[k / 2]);
        raw[k] = reinterpret_cast<const Raw*>(&r)[0];
        raw[k + 1] = reinterpret_cast<const Raw*>(&r)[1];
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        raw[k] = make_uint4(__float_as_uint(v[2 * k].x), __float_as_uint(v[2 * k].y), __float_as_uint(v[2 * k + 1].x),
                            __float_as_uint(v[2 * k + 1].y));
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
        raw[k] = make_uint4(pack_pair<T>(v[4 * k]), pack_pair<T>(v[4 * k + 1]), pack_pair<T>(v[4 * k + 2]), pack_pair<T>(v[4 * k + 3]));
    }
  }
};

// The threads that share a row: LANES of a warp, or (LANES = 0) whole warps, which meet at a barrier of their own.
struct RowTeam {
  int lanes, lane, group, groups;
};
template <int LANES>
__device__ __forceinline__ RowTeam row_team(const LayerNormParams& p) {
  RowTeam t;
  t.lanes = LANES ? LANES : p.lanes;
  t.lane = threadIdx.x % t.lanes;
  t.group = threadIdx.x / t.lanes;
  t.groups = blockDim.x / t.lanes;
  return t;
}

// Rows that are on their way: every thread copies its pieces of the next kDepth rows of N tensors into slots of its own in
// shared memory, asynchronously, and reads them back when it gets to the row; no other thread sees them, so there is no
// barrier. Loads into registers two and four rows ahead did not do: waiting for one of them waits for all behind it
// (forward, 32768 rows of 4096: 195 us that way, 97 this way). 16-bit rows of single elements and the widest ones are loaded
// directly.
template <typename T, bool WIDE, int K, int N>
struct RowsAhead {
  using Regs = RowRegs<T, WIDE, K>;
  static constexpr int kElements = K * Regs::V, kPiece = WIDE ? 16 : 4, kBytes = kPiece * K;
  static constexpr bool kStaged = (WIDE || sizeof(T) == 4) && kElements <= 32 && kElements * sizeof(T) * N <= 256;
  static constexpr int kDepth = !kStaged ? 1 : kElements <= 8 ? 4 : kElements * sizeof(T) <= 32 ? 3 : kElements * sizeof(T) <= 64 && (kElements < 32 || N < 3) ? 2 : 1;
  uint32_t slot;  // of this thread, in the stage that comes next
  uint32_t first, last, stage;

  __device__ __forceinline__ explicit RowsAhead(void* shared) {
    first = slot = static_cast<uint32_t>(__cvta_generic_to_shared(shared)) + threadIdx.x * kPiece;
    stage = blockDim.x * kBytes * N;
    last = first + (kDepth - 1) * stage;
  }
  // Starts the copies of a row of tensor n into the stage that comes next. `after`: behind what this value comes from.
  __device__ __forceinline__ void start(int n, const char* row, const RowTeam& t, int d, bool in, float after) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * t.lanes + t.lane) * Regs::V;
      const bool ok = in && c < d;
      const uint32_t to = slot + (n * K + k) * blockDim.x * kPiece;
      const char* from = ok ? row + c * static_cast<int>(sizeof(T)) : row;
      if constexpr (WIDE)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(ok ? 16 : 0), "f"(after) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(ok ? 4 : 0), "f"(after) : "memory");
    }
  }
  __device__ __forceinline__ void next() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    slot = slot == last ? first : slot + stage;
  }
  __device__ __forceinline__ void arrived() const { asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory"); }
  __device__ __forceinline__ void take(int n, Regs& r) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if constexpr (WIDE)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.raw[k].x), "=r"(r.raw[k].y), "=r"(r.raw[k].z), "=r"(r.raw[k].w)
                     : "r"(slot + (n * K + k) * blockDim.x * kPiece)
                     : "memory");
      else if constexpr (sizeof(T) == 4)
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r.raw[k]) : "r"(slot + (n * K + k) * blockDim.x * kPiece) : "memory");
  }
};

// The weights (or biases) of a lane's columns, of the rows' type or fp32; `none` where there are none. In registers for
// all rows where they are few, else read, from L1, for each row.
template <typename T, bool WIDE, int K>
struct LaneWeights {
  using Regs = RowRegs<T, WIDE, K>;
  static constexpr int V = Regs::V, kPairs = Regs::kPairs;
  static constexpr bool kKept = K * V <= 16;
  float2 v[kKept ? kPairs : 1];
  const char* p;
  int wide;
  float none;

  __device__ __forceinline__ LaneWeights(const void* weights, int w_wide, float if_none, int head, int lane, int lanes, int d) {
    wide = w_wide || sizeof(T) == 4;
    p = static_cast<const char*>(weights);
    if (p != nullptr) p += static_cast<long long>(head) * d * (wide ? 4 : 2);
    none = if_none;
    if constexpr (kKept) fetch(v, lane, lanes, d);
  }
  __device__ __forceinline__ void fetch(float2 (&w)[kPairs], int lane, int lanes, int d) const {
    if (p == nullptr) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) w[i] = make_float2(none, none);
    } else if (!wide) {
      Regs r;
      r.load(p, lane, lanes, d, true);
      r.widen(w);
    } else if constexpr (!WIDE) {
      RowRegs<float, false, K> r;
      r.load(p, lane, lanes, d, true);
      r.widen(w);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * lanes + lane) * V;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 q = c < d ? __ldg(reinterpret_cast<const float4*>(p + (c + i) * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
          w[(k * V + i) / 2] = make_float2(q.x, q.y);
          w[(k * V + i) / 2 + 1] = make_float2(q.z, q.w);
        }
      }
    }
  }
  __device__ __forceinline__ void get(float2 (&w)[kPairs], int lane, int lanes, int d) const {
    if constexpr (kKept) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) w[i] = v[i];
    } else {
      fetch(w, lane, lanes, d);
    }
  }
};

// Sums of N values over a row, the same in all of its threads. `parts`, of 32 words a value and turn for all groups
// together, alternates between two turns, so that one barrier a sum is enough.
template <int LANES, int N>
__device__ __forceinline__ void sum_over_row(float (&v)[N], float (*parts)[N][32], int& turn, const RowTeam& t) {
  constexpr int kSpan = LANES ? LANES : 32;
#pragma unroll
  for (int o = kSpan / 2; o > 0; o /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (LANES == 0) {
    const int warp = threadIdx.x / 32, warps = t.lanes / 32;
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) parts[turn][i][warp] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(t.group + 1), "r"(t.lanes) : "memory");
    const int w = threadIdx.x % 16;  // (a row has 16 warps at most)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = w < warps ? parts[turn][i][t.group * warps + w] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    turn ^= 1;
  }
}

// 1 / sqrt(v): the fast instruction, off by 2^-22, and a Newton step on it, which brings that to a rounding or two.
__device__ __forceinline__ float reciprocal_root(float v) {
  const float r = rsqrtf(v);
  return v > 0.f && v < 3e38f ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Registers decide how many threads an SM holds: up to 8 elements of a row a thread leave room for 1024 (backward, with
// two rows in fp32 at a time and the sums of the weights' gradients, 768), more for 512.
__host__ __device__ constexpr int norm_threads_sm(bool backward, int values) { return values > 8 ? 512 : backward ? 768 : 1024; }
__host__ __device__ constexpr int norm_threads_cta(bool backward, int values) { return values <= 8 && backward ? 256 : 512; }

// The next rows are on their way while these are worked on.
template <typename T, bool WIDE, int LANES, int K, bool FLAT>
__global__ void __launch_bounds__(norm_threads_cta(false, K * Piece<T, WIDE>::kElements), norm_threads_sm(false, K * Piece<T, WIDE>::kElements) / norm_threads_cta(false, K * Piece<T, WIDE>::kElements))
fla_layer_norm_fwd_kernel(const LayerNormParams p) {
  using Regs = RowRegs<T, WIDE, K>;
  constexpr int V = Regs::V, P = Regs::kPairs;
  // Two rows at a time share the latency of shuffles and barriers.
  constexpr int kRows = RowsAhead<T, WIDE, K, 2>::kStaged && K * V <= 8 ? 2 : 1;
  __shared__ float parts[2][kRows][32];
  int turn = 0;
  const RowTeam t = row_team<LANES>(p);
  const int head = blockIdx.y;
  const unsigned rows = static_cast<unsigned>(p.rows), stride = gridDim.x * t.groups;
  const float over_d = 1.f / p.d;
  const bool whole = t.lanes * K * V == p.d;  // no thread has pieces past the row
  const LaneWeights<T, WIDE, K> weight(p.w, p.w_wide, 1.f, head, t.lane, t.lanes, p.d), bias(p.b, p.w_wide, 0.f, head, t.lane, t.lanes, p.d);
  extern __shared__ uint4 slots[];
  using Ahead = RowsAhead<T, WIDE, K, 2>;
  Ahead ahead(slots);
  constexpr int R = kRows;
  Regs x[R], z[R];
  unsigned next = blockIdx.x * t.groups + t.group;
  Cursor<FLAT> x_at(p.x, head, next, stride), z_at(p.z, head, next, stride), s_at(p.s, head, next, stride), y_at(p.y, head, next, stride);
  auto fetch = [&](int r, float after) {  // the row after those that are on their way
    const bool in = next < rows;
    const char *xr = x_at.get(p, next, in), *zr = z_at.get(p, next, in && p.z.ptr != nullptr);
    if constexpr (Ahead::kStaged) {
      ahead.start(0, xr, t, p.d, in, after);
      if (p.z.ptr != nullptr) ahead.start(1, zr, t, p.d, in, after);
      ahead.next();
    } else {
      x[r].load(xr, t.lane, t.lanes, p.d, in);
      if (p.z.ptr != nullptr) z[r].load(zr, t.lane, t.lanes, p.d, in);
    }
    x_at.advance();
    z_at.advance();
    next += stride;
  };
#pragma unroll
  for (int s = 0; s < Ahead::kDepth; ++s) fetch(0, 0.f);
  unsigned j = blockIdx.x * t.groups + t.group;
  // (every lane of a warp takes the same turns: its first row decides)
  for (unsigned base = blockIdx.x * t.groups; base < rows; base += R * stride, j += R * stride) {
    float2 v[R][P];
    float sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned row = j + r * stride;
      if constexpr (Ahead::kStaged) {
        ahead.arrived();
        ahead.take(0, x[r]);
        if (p.z.ptr != nullptr) ahead.take(1, z[r]);
      }
      if (p.z.ptr != nullptr) {
        float2 more[P];
        x[r].widen(v[r]);
        z[r].widen(more);
#pragma unroll
        for (int i = 0; i < P; ++i) v[r][i] = add2(v[r][i], more[i]);
        x[r].narrow(v[r]);  // what is normalised is the sum as it is stored
        x[r].store(s_at.get(p, row, row < rows), t.lane, t.lanes, p.d, row < rows);
        s_at.advance();
      }
      x[r].widen(v[r]);
      float2 pair = v[r][0];
#pragma unroll
      for (int i = 1; i < P; ++i) pair = add2(pair, v[r][i]);
      sum[r] = pair.x + pair.y;
      fetch(r, sum[r]);
    }
    sum_over_row<LANES>(sum, parts, turn, t);
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = sum[r] * over_d;
#pragma unroll
      for (int i = 0; i < P; ++i) v[r][i] = add2(v[r][i], both(-mean[r]));
      if (!whole) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if ((2 * i / V * t.lanes + t.lane) * V >= p.d) v[r][i].x = 0.f;
          if (((2 * i + 1) / V * t.lanes + t.lane) * V >= p.d) v[r][i].y = 0.f;
        }
      }
      float2 pair = mul2(v[r][0], v[r][0]);
#pragma unroll
      for (int i = 1; i < P; ++i) pair = fma2(v[r][i], v[r][i], pair);
      sum[r] = pair.x + pair.y;
    }
    sum_over_row<LANES>(sum, parts, turn, t);
    float2 w[P], b[P];
    weight.get(w, t.lane, t.lanes, p.d);
    bias.get(b, t.lane, t.lanes, p.d);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned row = j + r * stride;
      const float root = reciprocal_root(fmaf(sum[r], over_d, p.eps));
      if (p.stats != nullptr && t.lane == 0 && row < rows)
        *reinterpret_cast<float2*>(stats_of<FLAT>(p, head, row)) = make_float2(mean[r], root);
#pragma unroll
      for (int i = 0; i < P; ++i) v[r][i] = fma2(mul2(v[r][i], both(root)), w[i], b[i]);
      Regs y;
      y.narrow(v[r]);
      y.store(y_at.get(p, row, row < rows), t.lane, t.lanes, p.d, row < rows);
      y_at.advance();
    }
  }
}

template <typename T, bool WIDE, int LANES, int K, bool FLAT>
__global__ void __launch_bounds__(norm_threads_cta(true, K * Piece<T, WIDE>::kElements), norm_threads_sm(true, K * Piece<T, WIDE>::kElements) / norm_threads_cta(true, K * Piece<T, WIDE>::kElements))
fla_layer_norm_bwd_kernel(const LayerNormParams p) {
  using Regs = RowRegs<T, WIDE, K>;
  constexpr int V = Regs::V, P = Regs::kPairs;
  __shared__ float parts[2][2][32];
  int turn = 0;
  const RowTeam t = row_team<LANES>(p);
  const int head = blockIdx.y;
  const unsigned rows = static_cast<unsigned>(p.rows), stride = gridDim.x * t.groups;
  const float over_d = 1.f / p.d;
  const LaneWeights<T, WIDE, K> weight(p.w, p.w_wide, 1.f, head, t.lane, t.lanes, p.d);
  // The sums for the weights: in registers, or, where 32 elements a thread leave none, in shared memory behind the rows.
  constexpr bool kSumsShared = WIDE && K * V == 32;
  float2 dw[kSumsShared ? 1 : P], db[kSumsShared ? 1 : P];
#pragma unroll
  for (int i = 0; i < (kSumsShared ? 1 : P); ++i) dw[i] = db[i] = both(0.f);
  extern __shared__ uint4 slots[];  // rows on their way; then [2][d] sums, where a CTA has several rows at a time
  using Ahead = RowsAhead<T, WIDE, K, 3>;
  Ahead ahead(slots);
  Regs x, dy, ds;
  float2 stats;
  const unsigned start = blockIdx.x * t.groups + t.group;
  unsigned next = start, stats_next = start;
  Cursor<FLAT> x_at(p.x, head, start, stride), dy_at(p.dy, head, start, stride), ds_at(p.ds, head, start, stride), dx_at(p.dx, head, start, stride);
  auto fetch = [&](float after) {  // the row after those that are on their way
    const bool in = next < rows;
    const char *xr = x_at.get(p, next, in), *gr = dy_at.get(p, next, in);
    if constexpr (Ahead::kStaged) {
      ahead.start(0, xr, t, p.d, in, after);
      ahead.start(1, gr, t, p.d, in, after);
      if (p.ds.ptr != nullptr) ahead.start(2, ds_at.get(p, next, in), t, p.d, in, after);
      ds_at.advance();
      ahead.next();
    } else {
      x.load(xr, t.lane, t.lanes, p.d, in);
      dy.load(gr, t.lane, t.lanes, p.d, in);
    }
    x_at.advance();
    dy_at.advance();
    next += stride;
  };
  auto fetch_stats = [&] {
    stats = stats_next < rows ? __ldg(reinterpret_cast<const float2*>(stats_of<FLAT>(p, head, stats_next))) : both(0.f);
    stats_next += stride;
  };
  float2* const sums_at = reinterpret_cast<float2*>(reinterpret_cast<char*>(slots) + (Ahead::kStaged ? 3 * Ahead::kDepth * Ahead::kBytes * blockDim.x : 0)) + threadIdx.x;
  if constexpr (kSumsShared)
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) sums_at[i * blockDim.x] = both(0.f);
  fetch_stats();
#pragma unroll
  for (int s = 0; s < Ahead::kDepth; ++s) fetch(0.f);
  unsigned j = start;
  for (unsigned base = blockIdx.x * t.groups; base < rows; base += stride, j += stride) {
    const bool in = j < rows;
    if constexpr (Ahead::kStaged) {
      ahead.arrived();
      ahead.take(0, x);
      ahead.take(1, dy);
      if (p.ds.ptr != nullptr) ahead.take(2, ds);
    } else {
      if (p.ds.ptr != nullptr) ds.load(ds_at.get(p, j, in), t.lane, t.lanes, p.d, in);
      ds_at.advance();
    }
    const float r = stats.y;
    const float2 shift = both(-stats.x);
    // (where there is no row, dy and r are zero, and past the end of a row dy: nothing is added)
    float2 n[P], u[P], w[P];
    x.widen(n);
    dy.widen(u);
    fetch_stats();
    weight.get(w, t.lane, t.lanes, p.d);
    float2 s0 = both(0.f), s1 = s0;  // of u and of u n
#pragma unroll
    for (int i = 0; i < P; ++i) {
      n[i] = mul2(add2(n[i], shift), both(r));
      if constexpr (kSumsShared) {
        float2* const at = sums_at + 2 * i * blockDim.x;
        at[0] = fma2(u[i], n[i], at[0]);
        at[blockDim.x] = add2(at[blockDim.x], u[i]);
      } else {
        dw[i] = fma2(u[i], n[i], dw[i]);
        db[i] = add2(db[i], u[i]);
      }
      u[i] = mul2(u[i], w[i]);
      s0 = add2(s0, u[i]);
      s1 = fma2(u[i], n[i], s1);
    }
    float sums[2] = {s0.x + s0.y, s1.x + s1.y};
    fetch(sums[1]);
    if (p.dx.ptr == nullptr) continue;
    sum_over_row<LANES>(sums, parts, turn, t);
    const float2 mean_u = both(-sums[0] * over_d), mean_un = both(-sums[1] * over_d);
#pragma unroll
    for (int i = 0; i < P; ++i) u[i] = mul2(fma2(n[i], mean_un, add2(u[i], mean_u)), both(r));
    if (p.ds.ptr != nullptr) {
      ds.widen(w);
#pragma unroll
      for (int i = 0; i < P; ++i) u[i] = add2(u[i], w[i]);
    }
    Regs dx;
    dx.narrow(u);
    dx.store(dx_at.get(p, j, in), t.lane, t.lanes, p.d, in);
    dx_at.advance();
  }
  if (p.parts == nullptr) return;
  asm volatile("griddepcontrol.launch_dependents;");  // (the kernel that joins the CTAs' sums may be set up)
  float* out = p.parts + (static_cast<long long>(blockIdx.x) * 2 * p.heads + head) * p.d;  // dw; db lies heads * d behind
  const long long db_at = static_cast<long long>(p.heads) * p.d;
  if constexpr (kSumsShared) {  // (one row at a time: every thread has columns of its own)
#pragma unroll
    for (int e = 0; e < 2 * P; ++e) {
      const int c = (e / V * t.lanes + t.lane) * V + e % V;
      const float2 ew = sums_at[2 * (e / 2) * blockDim.x], eb = sums_at[(2 * (e / 2) + 1) * blockDim.x];
      if (c < p.d) {
        out[c] = e % 2 ? ew.y : ew.x;
        out[db_at + c] = e % 2 ? eb.y : eb.x;
      }
    }
    return;
  } else {
  // The groups of a warp join by shuffles, then warps or groups of warps one after the other.
  constexpr int kSpan = LANES ? 32 : 0;
  float* const joined = reinterpret_cast<float*>(slots);
  if constexpr (Ahead::kStaged) asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();  // (the slots are free)
  if constexpr (LANES != 0)
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int o = LANES; o < 32; o *= 2) {
        dw[i] = add2(dw[i], make_float2(__shfl_xor_sync(0xffffffffu, dw[i].x, o), __shfl_xor_sync(0xffffffffu, dw[i].y, o)));
        db[i] = add2(db[i], make_float2(__shfl_xor_sync(0xffffffffu, db[i].x, o), __shfl_xor_sync(0xffffffffu, db[i].y, o)));
      }
  const int team = kSpan ? threadIdx.x / 32 : t.group, teams = kSpan ? static_cast<int>(blockDim.x) / 32 : t.groups;
  for (int turn_of = 0; turn_of < teams; ++turn_of) {
    if (team == turn_of && (LANES == 0 || threadIdx.x % 32 < LANES)) {
      float* const w_to = teams > 1 ? joined : out;
      float* const b_to = teams > 1 ? joined + p.d : out + db_at;
#pragma unroll
      for (int e = 0; e < 2 * P; ++e) {
        const int c = (e / V * t.lanes + t.lane) * V + e % V;
        const float ew = e % 2 ? dw[e / 2].y : dw[e / 2].x, eb = e % 2 ? db[e / 2].y : db[e / 2].x;
        if (c < p.d) {
          w_to[c] = turn_of ? w_to[c] + ew : ew;
          b_to[c] = turn_of ? b_to[c] + eb : eb;
        }
      }
    }
    __syncthreads();
  }
  if (teams > 1)
    for (int c = threadIdx.x; c < p.d; c += blockDim.x) {
      out[c] = joined[c];
      out[db_at + c] = joined[p.d + c];
    }
  }
}

// dw and db from the CTAs' sums: 32 columns a block, 32 shares of the CTAs side by side, joined in order.
template <typename W>
__global__ void __launch_bounds__(1024) fla_layer_norm_weights_kernel(const float* parts, int ctas, int columns, W* dw, W* db) {
  __shared__ float shares[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, share = threadIdx.y;
  W* out = blockIdx.y ? db : dw;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float sum = 0.f;
  const float* at = parts + static_cast<long long>(blockIdx.y) * columns + c;
  for (int i = share; i < ctas && c < columns; i += 32 * 8) {
    float some[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) some[k] = i + 32 * k < ctas ? __ldcg(at + static_cast<long long>(i + 32 * k) * 2 * columns) : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += some[k];
  }
  shares[share][threadIdx.x] = sum;
  __syncthreads();
  // a warp a column now
  sum = shares[threadIdx.x][share];
#pragma unroll
  for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int mine = blockIdx.x * 32 + share;
  if (threadIdx.x == 0 && mine < columns && out != nullptr) {
    if constexpr (sizeof(W) == 4) out[mine] = sum;
    else out[mine] = static_cast<W>(sum);
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
  int lanes, k;       // lanes: 0 where a row has whole warps, p.lanes threads
  int threads, ctas;  // ctas: of a head
  bool flat;
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

fla::Divisor divisor(int d) {
  unsigned l = 0;
  while ((1LL << l) < d) ++l;
  return {static_cast<unsigned>(d), static_cast<unsigned>((1ULL << (31 + l)) / d + 1), 31 + l};
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
  long long n0 = a->batch;
  // Rows are numbered as they lie in memory in what is normalised.
  const NormRows order = backward || p.s.ptr == nullptr ? p.x : p.s;
  p.stat_step[0] = p.n1 * p.n2;
  p.stat_step[1] = p.n2;
  p.stat_step[2] = 1;
  bool moved = false;  // a dim of several rows before another
  auto swap01 = [&] {
    moved = moved || (n0 > 1 && p.n1 > 1);
    std::swap(p.stat_step[0], p.stat_step[1]);
    for (NormRows* t : used) std::swap(t->s0, t->s1);
    const int n = static_cast<int>(n0);
    n0 = p.n1;
    p.n1 = n;
  };
  auto swap12 = [&] {
    moved = moved || (p.n1 > 1 && p.n2 > 1);
    std::swap(p.stat_step[1], p.stat_step[2]);
    for (NormRows* t : used) std::swap(t->s1, t->s2);
    std::swap(p.n1, p.n2);
  };
  {
    long long s0 = n0 == 1 ? 0 : order.s0, s1 = p.n1 == 1 ? 0 : order.s1, s2 = p.n2 == 1 ? 0 : order.s2;
    if (s1 > s0) swap01(), std::swap(s0, s1);
    if (s2 > s1) swap12(), std::swap(s1, s2);
    if (s1 > s0) swap01();
  }
  p.stat_n1 = divisor(p.n1);
  p.stat_n2 = divisor(p.n2);
  // neighbouring dims that are one in every tensor
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
  p.by_n1 = divisor(p.n1);
  p.by_n2 = divisor(p.n2);
  plan.flat = !moved && p.n1 == 1 && p.rows == p.n2;
  auto aligned = [](const void* q, int n) { return reinterpret_cast<uintptr_t>(q) % n == 0; };
  plan.wide = p.d % per == 0 && aligned(p.w, 16) && aligned(p.b, 16) && every([&](const NormRows& t) {
                return aligned(t.ptr, 16) && (p.heads == 1 || t.sh % 16 == 0) && (n0 == 1 || t.s0 % 16 == 0) &&
                       (p.n1 == 1 || t.s1 % 16 == 0) && (p.n2 == 1 || t.s2 % 16 == 0);
              });
  // A thread holds up to 16 elements of a row, 8 of the narrowest and 32 or 64 of the widest.
  const int pieces = plan.wide ? p.d / per : p.d;
  const int held = plan.wide ? per : 1;
  const int values = p.d <= 32 ? 8 : p.d <= 8192 ? 16 : p.d <= 16384 ? 32 : 64;
  plan.k = values / held;
  if (!plan.wide) plan.k = p.d <= 64 ? 2 : p.d <= 128 ? 4 : p.d <= 256 ? 8 : plan.k;
  plan.lanes = plan.wide && pieces <= 4 * plan.k ? 4 : plan.wide && pieces <= 8 * plan.k ? 8 : plan.wide && pieces <= 16 * plan.k ? 16 : pieces <= 32 * plan.k ? 32 : 0;
  p.lanes = plan.lanes ? plan.lanes : (pieces + plan.k * 32 - 1) / (plan.k * 32) * 32;
  const long long groups = std::max(1, 256 / p.lanes);
  plan.threads = static_cast<int>(groups) * p.lanes;
  // As many CTAs as are resident together; a CTA of the backward leaves a row of sums behind, so it has two turns or more.
  const int resident = std::max(1, fla::norm_threads_sm(backward, plan.k * held) / plan.threads);
  const long long most = std::max<long long>(1, static_cast<long long>(sm_count) * resident / p.heads);
  const long long turns = (p.rows + groups - 1) / groups;
  plan.ctas = static_cast<int>(std::min(most, backward ? (turns + 1) / 2 : turns));
  return plan;
}

size_t norm_workspace(const NormPlan& plan) { return static_cast<size_t>(plan.ctas) * 2 * plan.p.heads * plan.p.d * sizeof(float); }

template <typename T, bool WIDE, int LANES, int K, bool FLAT>
int norm_launch_kernel(const NormPlan& plan, bool backward, cudaStream_t stream) {
  using Forward = fla::RowsAhead<T, WIDE, K, 2>;
  using Backward = fla::RowsAhead<T, WIDE, K, 3>;
  const dim3 grid(plan.ctas, plan.p.heads);
  const auto kernel = backward ? fla::fla_layer_norm_bwd_kernel<T, WIDE, LANES, K, FLAT>
                               : fla::fla_layer_norm_fwd_kernel<T, WIDE, LANES, K, FLAT>;
  // (the stages are laid out for the most tensors that a row can have)
  size_t shared = static_cast<size_t>(plan.threads) * (backward ? Backward::kStaged * Backward::kDepth * Backward::kBytes * 3
                                                                : Forward::kStaged * Forward::kDepth * Forward::kBytes * 2);
  constexpr int kElements = Backward::kElements;
  if (backward && WIDE && kElements == 32) shared += 2 * kElements * plan.threads * sizeof(float);
  else if (backward && plan.p.parts != nullptr && plan.threads > std::max(32, plan.p.lanes))
    shared = std::max(shared, 2 * plan.p.d * sizeof(float));
  if (shared > 40 * 1024 &&  // (48 KB go without, with what the kernels declare)
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)) != cudaSuccess)
    return FLA_ERR_CUDA;
  kernel<<<grid, plan.threads, shared, stream>>>(plan.p);
  return fla::launched(cudaSuccess, backward ? "fla_layer_norm_bwd_kernel" : "fla_layer_norm_fwd_kernel");
}

template <typename T, bool WIDE, int LANES, int K>
int norm_launch(const NormPlan& plan, bool backward, cudaStream_t stream) {
  // Long 16-bit rows of single elements, which are not staged, gain nothing from advanced addresses: backward, with and without,
  // 16384 x 1023 in bf16 101 and 52 us, 8192 x 4099 in fp16 with a residual 402 and 175 (forward 35 and 34, 132 and 128). All
  // others do: 65536 x 83 in bf16 19 and 26 forward, 29 and 36 backward; 32768 x 4096 with a residual 179 and 191 backward.
  if constexpr (!WIDE && LANES == 0 && sizeof(T) == 2)
    return norm_launch_kernel<T, WIDE, LANES, K, false>(plan, backward, stream);
  else
    return plan.flat ? norm_launch_kernel<T, WIDE, LANES, K, true>(plan, backward, stream)
                     : norm_launch_kernel<T, WIDE, LANES, K, false>(plan, backward, stream);
}

template <typename T>
int norm_launch_type(const NormPlan& plan, bool backward, cudaStream_t stream) {
  constexpr int kPer = 16 / sizeof(T), k8 = 8 / kPer;  // elements of a piece, pieces of 8 elements
  if (plan.wide) {
    if (plan.k == k8) return norm_launch<T, true, 4, k8>(plan, backward, stream);
    if (plan.lanes == 4) return norm_launch<T, true, 4, 2 * k8>(plan, backward, stream);
    if (plan.lanes == 8) return norm_launch<T, true, 8, 2 * k8>(plan, backward, stream);
    if (plan.lanes == 16) return norm_launch<T, true, 16, 2 * k8>(plan, backward, stream);
    if (plan.lanes == 32) return norm_launch<T, true, 32, 2 * k8>(plan, backward, stream);
    if (plan.k == 2 * k8) return norm_launch<T, true, 0, 2 * k8>(plan, backward, stream);
    if (plan.k == 4 * k8) return norm_launch<T, true, 0, 4 * k8>(plan, backward, stream);
    return norm_launch<T, true, 0, 8 * k8>(plan, backward, stream);
  }
  if (plan.lanes && plan.k == 2) return norm_launch<T, false, 32, 2>(plan, backward, stream);
  if (plan.lanes && plan.k == 4) return norm_launch<T, false, 32, 4>(plan, backward, stream);
  if (plan.lanes && plan.k == 8) return norm_launch<T, false, 32, 8>(plan, backward, stream);
  if (plan.lanes) return norm_launch<T, false, 32, 16>(plan, backward, stream);
  if (plan.k == 16) return norm_launch<T, false, 0, 16>(plan, backward, stream);
  if (plan.k == 32) return norm_launch<T, false, 0, 32>(plan, backward, stream);
  return norm_launch<T, false, 0, 64>(plan, backward, stream);
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
  // Set up while the first kernel runs; it waits for that one's end (which is a launch's latency less, 3 us).
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((columns + 31) / 32, 2);
  cfg.blockDim = dim3(32, 32);
  cfg.stream = static_cast<cudaStream_t>(a->stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto go = [&](auto* zero) {
    using W = std::remove_pointer_t<decltype(zero)>;
    return fla::launched(cudaLaunchKernelEx(&cfg, fla::fla_layer_norm_weights_kernel<W>, static_cast<const float*>(plan.p.parts), plan.ctas,
                                            columns, static_cast<W*>(a->d_weight), static_cast<W*>(a->d_bias)),
                         "fla_layer_norm_weights_kernel");
  };
  if (a->w_dtype == FLA_DTYPE_F32) return go(static_cast<float*>(nullptr));
  if (a->w_dtype == FLA_DTYPE_F16) return go(static_cast<__half*>(nullptr));
  return go(static_cast<__nv_bfloat16*>(nullptr));
}

}  // extern "C"
