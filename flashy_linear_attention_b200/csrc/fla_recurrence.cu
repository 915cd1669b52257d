// Gated linear recurrence for sm_100a: every channel of a head carries a state of its own,
//     h_t = exp(g_t) h_(t-1) + x_t,      out_t = h_t,
// and with G_t = dO_t + R_(t+1), R_t = exp(g_t) G_t the gradients are
//     dx_t = G_t,   dg_t = R_t h_(t-1),  d(s_init) = R_0,  R_N = d(s_final).
// The reference has no counterpart (its mixers are products of q, k and v, flashlinear/linear_attn.py:11-31).
//
// Bound by HBM: two multiply-adds and an exp an element next to 6 bytes (16-bit rows; the backward 10). What it
// takes is that enough of a sequence is in flight although each step waits for the one before. A step is a map
// c -> a c + b, and the composition of steps is such a map again, so a run of T tokens is summed from zero
// (b) with its decay (a = exp of the sum of its g) without knowing what came before:
//   * a thread holds two channels of a run of T = 16 tokens (8 with fp32 rows) in registers, read once;
//   * the runs of a CTA exchange (a, b) through shared memory, the CTAs of a cluster, which share a tile of channels
//     and take neighbouring stretches of tokens, through distributed shared memory, both in one fixed order;
//   * then each run is walked again from the state before it, out of registers.
// A cluster walks its sequence from end to end, the rows of the next step being on their way while it
// exchanges. Nothing is read twice, there is no scratch, no atomic and no wait on memory, and the order of all sums
// depends on the shapes only.
//
// Accuracy. Channels with a memory of ten thousand tokens multiply the state by exp(-1e-4) as often. That
// factor rounded to 32 bits is off by up to 3e-8, every time in the same direction. The state is therefore multiplied
// once a run, by exp(sum of g) held as two floats; the decays of single tokens only act within a run.
//
// A gate of minus infinity (a document starts) drops the state whatever it holds, infinities and NaN included, and
// nothing flows back past it.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "fla_internal.h"
#include "fla_pairs.cuh"

namespace fla {

namespace cg = cooperative_groups;

struct RecurrenceTensor {
  void* ptr;
  long long sb, sh, sn;  // element strides; innermost stride 1
};

struct RecurrenceParams {
  RecurrenceTensor x, g, o;   // o: out (forward), dO (backward; ptr null: zero)
  RecurrenceTensor dx, dg;    // backward outputs (ptr null: not wanted)
  const float* start;         // [bh][c]: state before the first token (forward), R_N (backward); null: zero
  float* end;                 // [bh][c]: state after the last token, resp. R_0; null: not wanted
  float* states;              // [b][run][heads * c]: the state before each run; null: not wanted (forward)
  int heads, n, c;
  int tiles;                  // tiles of channels a (batch, head)
  long long tiles_all;
};

constexpr int kRecThreads = 256;
constexpr int kRecMaxCluster = 8;

// Tokens a thread holds: a run. 16-bit rows and gates leave room for twice as many.
template <typename TX, typename TG>
constexpr int kRunTokens = sizeof(TX) + sizeof(TG) <= 4 ? 16 : 8;

// The map of a run, c -> (hi + lo) c + b, for two channels. hi < 0: the run drops what came before.
struct RunMap {
  float2 hi, lo, b;
};

__device__ __forceinline__ float apply_map(float c, float hi, float lo, float b) {
  // (from zero the map is b, also where a growing gate has overflowed; the correction of an infinite state is NaN)
  if (hi < 0.f || c == 0.f) return b;
  return fmaf(hi, c, fabsf(c) <= 3.4e38f ? fmaf(lo, c, b) : b);
}
__device__ __forceinline__ float2 apply_map(float2 c, const RunMap& m) {
  return make_float2(apply_map(c.x, m.hi.x, m.lo.x, m.b.x), apply_map(c.y, m.hi.y, m.lo.y, m.b.y));
}

// A decay that would round to zero (the smallest normal number): what it adds is below 2^-126 of the state, but an
// infinity stays one until a gate of minus infinity, as it does token by token.
constexpr float kLeastDecay = 1.17549435e-38f;

// exp(s) as hi + lo. Near 1, where the error of one float would act on a long memory, the second takes up what the
// first lost: exp(s) - 1 from its series (s^7 / 5040 is below 2^-31 of it there).
__device__ __forceinline__ void split_exp(float s, float* hi, float* lo) {
  if (s == -INFINITY) {
    *hi = -1.f;
    *lo = 0.f;
    return;
  }
  float e = fmaf(s, 1.f / 720.f, 1.f / 120.f);
  e = fmaf(s, e, 1.f / 24.f);
  e = fmaf(s, e, 1.f / 6.f);
  e = fmaf(s, e, 0.5f);
  e = fmaf(s * s, e, s);
  const bool near = fabsf(s) < 0.125f;
  *hi = near ? 1.f + e : fmaxf(expf(s), kLeastDecay);
  *lo = near ? e - (*hi - 1.f) : 0.f;
}

// Decay of one token. 16-bit rows: the fast exponential, off by 2^-22 or so, which acts on 16 tokens at most.
template <typename TX>
__device__ __forceinline__ float decay(float g) {
  return sizeof(TX) == 4 ? expf(g) : __expf(g);
}
template <typename TX>
__device__ __forceinline__ float advance(float g, float h, float x) {
  return g == -INFINITY ? x : fmaf(decay<TX>(g), h, x);
}

// Composition: first m, then n.
__device__ __forceinline__ void then_map(float& hi, float& lo, float& b, float nhi, float nlo, float nb) {
  b = apply_map(b, nhi, nlo, nb);
  if (hi < 0.f || nhi < 0.f) {
    hi = -1.f;
    lo = 0.f;
    return;
  }
  const float p = hi * nhi;
  lo = fmaf(hi, nhi, -p) + fmaf(hi, nlo, lo * nhi);
  hi = fmaxf(p, kLeastDecay);
}

template <int LPR>
struct RecurrenceShared {
  RunMap run[2][kRecThreads];          // [step parity][run of the CTA][lane]
  RunMap cta[2][kRecMaxCluster][LPR];  // [step parity][CTA of the cluster][lane]
};
struct Nothing {};

struct Place {  // what a thread works on
  long long tile;
  int lane, run, runs, rank, ranks;
  int b, h, c0, gap;
  bool ok0, ok1;
};

// Exchanges the maps of a step. `carry` is the state before the cluster's step and becomes the one behind it; returns
// the state before this thread's run. `order`: position of the run among the CTA's, of the CTA among the cluster's, in
// the direction of the walk.
template <int LPR>
__device__ __forceinline__ float2 exchange(RecurrenceShared<LPR>& sh, int parity, const RunMap& mine, const Place& w,
                                           float2& carry) {
  const int run = w.run, runs = w.runs, lane = w.lane, rank = w.rank, ranks = w.ranks;
  RunMap* maps = sh.run[parity];
  maps[run * LPR + lane] = mine;
  __syncthreads();
  float2 c = carry, before = carry;
  if (ranks == 1) {
#pragma unroll 4
    for (int r = 0; r < runs; ++r) {
      if (r == run) before = c;
      c = apply_map(c, maps[r * LPR + lane]);
    }
    carry = c;
    return before;
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (run == 0) {
    RunMap all = maps[lane];
    for (int r = 1; r < runs; ++r) {
      const RunMap m = maps[r * LPR + lane];
      then_map(all.hi.x, all.lo.x, all.b.x, m.hi.x, m.lo.x, m.b.x);
      then_map(all.hi.y, all.lo.y, all.b.y, m.hi.y, m.lo.y, m.b.y);
    }
    for (int r = 0; r < ranks; ++r)  // (cluster ranks and the order of the walk are the same)
      *cluster.map_shared_rank(&sh.cta[parity][rank][lane], r) = all;
  }
  // A CTA overwrites what it wrote two steps ago, which its peers have read before they came to the barrier of the step
  // between; after the last barrier nobody writes to a peer, so a CTA may leave.
  cluster.sync();
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) before = c;
    c = apply_map(c, sh.cta[parity][r][lane]);
  }
  carry = c;
  c = before;
  for (int r = 0; r < run; ++r) c = apply_map(c, maps[r * LPR + lane]);
  return c;
}

// ALONE: every group of LPR lanes has a tile and all its tokens to itself (short sequences: nothing to exchange).
template <bool PAIR, int LPR, bool ALONE>
__device__ __forceinline__ Place place(const RecurrenceParams& p) {
  Place w;
  w.lane = threadIdx.x % LPR;
  const int group = threadIdx.x / LPR, groups = blockDim.x / LPR;
  if (ALONE) {
    w.run = w.rank = 0;
    w.runs = w.ranks = 1;
    w.tile = static_cast<long long>(blockIdx.x) * groups + group;
  } else {
    cg::cluster_group cluster = cg::this_cluster();
    w.run = group;
    w.runs = groups;
    w.ranks = cluster.num_blocks();
    w.rank = cluster.block_rank();
    w.tile = blockIdx.x / w.ranks;
  }
  const long long bh = w.tile / p.tiles;
  w.b = static_cast<int>(bh / p.heads);
  w.h = static_cast<int>(bh % p.heads);
  w.gap = PAIR ? 1 : LPR;
  w.c0 = static_cast<int>(w.tile % p.tiles) * 2 * LPR + (PAIR ? 2 * w.lane : w.lane);
  w.ok0 = w.c0 < p.c && w.tile < p.tiles_all;
  w.ok1 = w.c0 + w.gap < p.c && w.tile < p.tiles_all;
  return w;
}

// Index into RecurrenceParams::states, whose layout does not depend on how heads were joined.
__device__ __forceinline__ long long state_of(const RecurrenceParams& p, const Place& w, int run, int runs_all) {
  return ((static_cast<long long>(w.b) * runs_all + run) * p.heads + w.h) * p.c + w.c0;
}

template <typename T>
__device__ __forceinline__ T* row0(const RecurrenceTensor& t, const Place& w) {
  return static_cast<T*>(t.ptr) + w.b * t.sb + w.h * t.sh + w.c0;
}

template <typename TX, typename TG, bool PAIR, int LPR, bool ALONE>
__global__ void __launch_bounds__(kRecThreads, 2) fla_recurrence_fwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  __shared__ std::conditional_t<ALONE, Nothing, RecurrenceShared<LPR>> sh;
  const Place w = place<PAIR, LPR, ALONE>(p);
  if (ALONE && !w.ok0) return;
  const TX* xp = row0<const TX>(p.x, w);
  const TG* gp = row0<const TG>(p.g, w);
  TX* op = row0<TX>(p.o, w);
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  if (p.start != nullptr) carry = load_pair<float, PAIR>(p.start + cell, w.gap, w.ok0, w.ok1);

  typename PairOf<TX>::Raw x[T], x_next[T];
  typename PairOf<TG>::Raw g[T], g_next[T];
  const int span = w.ranks * w.runs * T;  // tokens a step
  const int steps = (p.n - 1) / span + 1;
  auto fetch = [&](int t0, auto& xr, auto& gr) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const bool in = t0 + t < p.n;
      xr[t] = load_pair<TX, PAIR>(xp + (t0 + t) * p.x.sn, w.gap, w.ok0 && in, w.ok1 && in);
      gr[t] = load_pair<TG, PAIR>(gp + (t0 + t) * p.g.sn, w.gap, w.ok0 && in, w.ok1 && in);
    }
  };
  const int first = (w.rank * w.runs + w.run) * T;
  fetch(first, x, g);
  if (!ALONE && w.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
  for (int step = 0; step < steps; ++step) {
    const int t0 = step * span + first;
    if (step + 1 < steps) fetch(t0 + span, x_next, g_next);
    float2 h = carry;
    if constexpr (!ALONE) {
      h = make_float2(0.f, 0.f);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float2 xv = unpack_pair<TX>(x[t]), gv = unpack_pair<TG>(g[t]);
        sum.x += gv.x;
        sum.y += gv.y;
        h.x = advance<TX>(gv.x, h.x, xv.x);
        h.y = advance<TX>(gv.y, h.y, xv.y);
      }
      RunMap m;
      m.b = h;
      split_exp(sum.x, &m.hi.x, &m.lo.x);
      split_exp(sum.y, &m.hi.y, &m.lo.y);
      h = exchange<LPR>(sh, step & 1, m, w, carry);
    }
    if (p.states != nullptr && t0 < p.n)
      store_pair<float, PAIR>(p.states + state_of(p, w, t0 / T, (p.n - 1) / T + 1), w.gap, w.ok0, w.ok1, h);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float2 xv = unpack_pair<TX>(x[t]), gv = unpack_pair<TG>(g[t]);
      if constexpr (ALONE) {  // (a program that decodes multiplies its state once a call, by one token's decay)
        RunMap m;
        m.b = xv;
        split_exp(gv.x, &m.hi.x, &m.lo.x);
        split_exp(gv.y, &m.hi.y, &m.lo.y);
        h = apply_map(h, m);
      } else {
        h.x = advance<TX>(gv.x, h.x, xv.x);
        h.y = advance<TX>(gv.y, h.y, xv.y);
      }
      const bool in = t0 + t < p.n;
      store_pair<TX, PAIR>(op + (t0 + t) * p.o.sn, w.gap, w.ok0 && in, w.ok1 && in, h);
    }
    if (ALONE) carry = h;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      x[t] = x_next[t];
      g[t] = g_next[t];
    }
  }
  if (p.end != nullptr && w.run == 0 && w.rank == 0) store_pair<float, PAIR>(p.end + cell, w.gap, w.ok0, w.ok1, carry);
}

template <typename TX, typename TG, bool PAIR, int LPR, bool ALONE>
__global__ void __launch_bounds__(kRecThreads, 2) fla_recurrence_bwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  __shared__ std::conditional_t<ALONE, Nothing, RecurrenceShared<LPR>> sh;
  const Place w = place<PAIR, LPR, ALONE>(p);
  if (ALONE && !w.ok0) return;
  const TX* xp = row0<const TX>(p.x, w);
  const TG* gp = row0<const TG>(p.g, w);
  const TX* yp = row0<const TX>(p.o, w);
  TX* dxp = row0<TX>(p.dx, w);
  TG* dgp = row0<TG>(p.dg, w);
  const bool has_dy = p.o.ptr != nullptr;
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  if (p.start != nullptr) carry = load_pair<float, PAIR>(p.start + cell, w.gap, w.ok0, w.ok1);

  const int runs_all = (p.n - 1) / T + 1;
  const int span = w.ranks * w.runs;  // runs a step
  if (!ALONE && w.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
  const int steps = (runs_all - 1) / span + 1;
  for (int step = 0; step < steps; ++step) {
    // the walk starts at the end; its first runs may lie behind the last token and are the identity
    const int run = steps * span - 1 - ((step * w.ranks + w.rank) * w.runs + w.run);
    const int t0 = run * T;
    typename PairOf<TX>::Raw x[T], y[T];
    typename PairOf<TG>::Raw g[T];
    float2 h = make_float2(0.f, 0.f);
    if (run < runs_all) h = load_pair<float, PAIR>(p.states + state_of(p, w, run, runs_all), w.gap, w.ok0, w.ok1);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const bool in = t0 + t < p.n;
      x[t] = load_pair<TX, PAIR>(xp + (t0 + t) * p.x.sn, w.gap, w.ok0 && in, w.ok1 && in);
      g[t] = load_pair<TG, PAIR>(gp + (t0 + t) * p.g.sn, w.gap, w.ok0 && in, w.ok1 && in);
      y[t] = load_pair<TX, PAIR>(yp + (t0 + t) * p.o.sn, w.gap, w.ok0 && in && has_dy, w.ok1 && in && has_dy);
    }
    float2 before[T];  // the state before each token
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float2 xv = unpack_pair<TX>(x[t]), gv = unpack_pair<TG>(g[t]);
      before[t] = h;
      h.x = advance<TX>(gv.x, h.x, xv.x);
      h.y = advance<TX>(gv.y, h.y, xv.y);
    }
    float2 r = carry;
    if constexpr (!ALONE) {
      r = make_float2(0.f, 0.f);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int t = T - 1; t >= 0; --t) {
        const float2 yv = unpack_pair<TX>(y[t]), gv = unpack_pair<TG>(g[t]);
        sum.x += gv.x;
        sum.y += gv.y;
        r.x = gv.x == -INFINITY ? 0.f : decay<TX>(gv.x) * (yv.x + r.x);
        r.y = gv.y == -INFINITY ? 0.f : decay<TX>(gv.y) * (yv.y + r.y);
      }
      RunMap m;
      m.b = r;
      split_exp(sum.x, &m.hi.x, &m.lo.x);
      split_exp(sum.y, &m.hi.y, &m.lo.y);
      r = exchange<LPR>(sh, step & 1, m, w, carry);
    }
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      const float2 yv = unpack_pair<TX>(y[t]), gv = unpack_pair<TG>(g[t]);
      const bool in = t0 + t < p.n;
      const float2 all = make_float2(yv.x + r.x, yv.y + r.y);
      if (p.dx.ptr != nullptr) store_pair<TX, PAIR>(dxp + (t0 + t) * p.dx.sn, w.gap, w.ok0 && in, w.ok1 && in, all);
      const bool drop0 = gv.x == -INFINITY, drop1 = gv.y == -INFINITY;
      r.x = drop0 ? 0.f : decay<TX>(gv.x) * all.x;
      r.y = drop1 ? 0.f : decay<TX>(gv.y) * all.y;
      if (p.dg.ptr != nullptr)
        store_pair<TG, PAIR>(dgp + (t0 + t) * p.dg.sn, w.gap, w.ok0 && in, w.ok1 && in,
                             make_float2(drop0 ? 0.f : r.x * before[t].x, drop1 ? 0.f : r.y * before[t].y));
    }
    if (ALONE) carry = r;
  }
  if (p.end != nullptr && w.run == 0 && w.rank == 0) store_pair<float, PAIR>(p.end + cell, w.gap, w.ok0, w.ok1, carry);
}

}  // namespace fla

namespace {

using fla::RecurrenceParams;
using fla::RecurrenceTensor;

constexpr int kAloneTokens = 32;  // sequences up to here have nothing to exchange

int element_bytes(int dtype) { return dtype == FLA_DTYPE_F32 ? 4 : 2; }

// The call as the kernels see it. Channels of all heads (and, for one token, of the batch) that lie next to each
// other in every tensor are one row: narrow heads then fill a warp.
struct Plan {
  RecurrenceParams p;
  bool pair;
  int lpr;
  int batch;
};

void add_tensor(const FlaTensor& t, RecurrenceTensor* out) {
  out->ptr = t.ptr;
  out->sb = t.stride_b;
  out->sh = t.stride_h;
  out->sn = t.stride_n;
}

Plan make_plan(const FlaRecurrenceArgs* a, bool backward) {
  Plan plan = {};
  RecurrenceParams& p = plan.p;
  add_tensor(a->x, &p.x);
  add_tensor(a->g, &p.g);
  add_tensor(backward ? a->d_o : a->o, &p.o);
  if (backward) {
    add_tensor(a->d_x, &p.dx);
    add_tensor(a->d_g, &p.dg);
  }
  p.start = backward ? a->r_init : a->s_init;
  p.end = backward ? a->r_final : a->s_final;
  p.states = static_cast<float*>(a->states);
  p.heads = a->heads;
  p.n = a->seqlen;
  p.c = a->dim;
  plan.batch = a->batch;
  RecurrenceTensor* const all[] = {&p.x, &p.g, &p.o, &p.dx, &p.dg};
  const int sizes[] = {element_bytes(a->dtype), element_bytes(a->g_dtype), element_bytes(a->dtype),
                       element_bytes(a->dtype), element_bytes(a->g_dtype)};
  auto every = [&](auto&& holds) {
    bool ok = true;
    for (int i = 0; i < 5; ++i)
      if (all[i]->ptr != nullptr) ok = ok && holds(*all[i], sizes[i]);
    return ok;
  };
  const long long wide = static_cast<long long>(p.heads) * p.c;
  if (p.heads > 1 && wide < (1 << 30) && every([&](const RecurrenceTensor& t, int) { return t.sh == p.c; })) {
    p.c = static_cast<int>(wide);
    p.heads = 1;
  }
  const long long flat = static_cast<long long>(plan.batch) * p.c;
  if (p.heads == 1 && p.n == 1 && plan.batch > 1 && flat < (1 << 30) &&
      every([&](const RecurrenceTensor& t, int) { return t.sb == p.c; })) {
    p.c = static_cast<int>(flat);
    plan.batch = 1;
  }
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 8 == 0; };
  plan.pair = p.c % 2 == 0 && aligned(p.start) && aligned(p.end) && aligned(p.states) &&
              every([&](const RecurrenceTensor& t, int size) {
                return reinterpret_cast<uintptr_t>(t.ptr) % (2 * size) == 0 && (p.n == 1 || t.sn % 2 == 0) &&
                       (p.heads == 1 || t.sh % 2 == 0) && (plan.batch == 1 || t.sb % 2 == 0);
              });
  plan.lpr = p.c <= 32 ? 16 : 32;
  p.tiles = (p.c + 2 * plan.lpr - 1) / (2 * plan.lpr);
  p.tiles_all = static_cast<long long>(p.tiles) * p.heads * plan.batch;
  return plan;
}

// CTAs of a cluster and threads of a CTA. A tile of channels is walked by one cluster from end to end; more CTAs walk
// it in fewer steps. Two CTAs are resident an SM.
void shape_of(const Plan& plan, int run_tokens, int sm_count, int* threads, int* ranks) {
  const long long runs = (plan.p.n - 1) / run_tokens + 1;
  int per_cta = 1;
  while (per_cta < fla::kRecThreads / plan.lpr && per_cta < runs) per_cta *= 2;
  int r = 1;
  while (r < fla::kRecMaxCluster && plan.p.tiles_all * r < 2 * sm_count && static_cast<long long>(r) * per_cta < runs) r *= 2;
  *threads = std::max(32, per_cta * plan.lpr);
  *ranks = r;
}

template <typename TX, typename TG, bool PAIR, int LPR, bool ALONE>
int launch(const Plan& plan, bool backward, int sm_count, cudaStream_t stream) {
  int threads = 128, ranks = 1;
  long long blocks;
  if (ALONE) {
    blocks = (plan.p.tiles_all * LPR + threads - 1) / threads;
  } else {
    shape_of(plan, fla::kRunTokens<TX, TG>, sm_count, &threads, &ranks);
    blocks = plan.p.tiles_all * ranks;
  }
  if (blocks > 0x7fffffffLL) return FLA_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  if (backward)
    return fla::launched(cudaLaunchKernelEx(&cfg, fla::fla_recurrence_bwd_kernel<TX, TG, PAIR, LPR, ALONE>, plan.p),
                         "fla_recurrence_bwd_kernel");
  return fla::launched(cudaLaunchKernelEx(&cfg, fla::fla_recurrence_fwd_kernel<TX, TG, PAIR, LPR, ALONE>, plan.p),
                       "fla_recurrence_fwd_kernel");
}

template <typename TX, typename TG>
int launch_types(const Plan& plan, bool backward, int sm_count, cudaStream_t stream) {
  const bool alone = plan.p.n <= kAloneTokens;
  auto pick = [&](auto pair, auto lpr) {
    constexpr bool P = decltype(pair)::value;
    constexpr int L = decltype(lpr)::value;
    return alone ? launch<TX, TG, P, L, true>(plan, backward, sm_count, stream)
                 : launch<TX, TG, P, L, false>(plan, backward, sm_count, stream);
  };
  using L16 = std::integral_constant<int, 16>;
  using L32 = std::integral_constant<int, 32>;
  if (plan.pair) return plan.lpr == 16 ? pick(std::true_type(), L16()) : pick(std::true_type(), L32());
  return plan.lpr == 16 ? pick(std::false_type(), L16()) : pick(std::false_type(), L32());
}

bool known_type(int t) { return t == FLA_DTYPE_BF16 || t == FLA_DTYPE_F16 || t == FLA_DTYPE_F32; }

int check(const FlaRecurrenceArgs* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->seqlen <= 0 || a->dim <= 0) return FLA_ERR_INVALID;
  if (!known_type(a->dtype) || (a->g_dtype != a->dtype && a->g_dtype != FLA_DTYPE_F32)) return FLA_ERR_INVALID;
  if (a->x.ptr == nullptr || a->g.ptr == nullptr) return FLA_ERR_INVALID;
  // run and token numbers are 32-bit, a step past the end included
  if (a->seqlen > (1 << 30) || static_cast<long long>(a->batch) * a->heads > (1 << 30)) return FLA_ERR_UNSUPPORTED;
  const int x = element_bytes(a->dtype), g = element_bytes(a->g_dtype);
  auto off = [](const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
  if (off(a->x.ptr, x) || off(a->o.ptr, x) || off(a->d_o.ptr, x) || off(a->d_x.ptr, x) || off(a->g.ptr, g) ||
      off(a->d_g.ptr, g) || off(a->s_init, 4) || off(a->s_final, 4) || off(a->r_init, 4) || off(a->r_final, 4) ||
      off(a->states, 16))
    return FLA_ERR_ALIGNMENT;
  return FLA_OK;
}

int run(const FlaRecurrenceArgs* a, bool backward) {
  (void)cudaGetLastError();
  fla::g_last_launches = 0;
  int sm_count = 0;
  if (const int rc = fla::block_device(&sm_count)) return rc;
  const Plan plan = make_plan(a, backward);
  cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
  const bool wide_gates = a->g_dtype == FLA_DTYPE_F32;
  if (a->dtype == FLA_DTYPE_F32) return launch_types<float, float>(plan, backward, sm_count, stream);
  if (a->dtype == FLA_DTYPE_F16)
    return wide_gates ? launch_types<__half, float>(plan, backward, sm_count, stream)
                      : launch_types<__half, __half>(plan, backward, sm_count, stream);
  return wide_gates ? launch_types<__nv_bfloat16, float>(plan, backward, sm_count, stream)
                    : launch_types<__nv_bfloat16, __nv_bfloat16>(plan, backward, sm_count, stream);
}

}  // namespace

extern "C" {

size_t fla_sm100_recurrence_states_bytes(const FlaRecurrenceArgs* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->seqlen <= 0 || a->dim <= 0) return 0;
  const int tokens = element_bytes(a->dtype) + element_bytes(a->g_dtype) <= 4 ? 16 : 8;
  const size_t runs = (static_cast<size_t>(a->seqlen) - 1) / tokens + 1;
  return runs * a->batch * a->heads * a->dim * sizeof(float);
}

int fla_sm100_recurrence_fwd(const FlaRecurrenceArgs* a) {
  if (const int rc = check(a)) return rc;
  if (a->o.ptr == nullptr) return FLA_ERR_INVALID;
  if (a->states != nullptr && a->states_bytes < fla_sm100_recurrence_states_bytes(a)) return FLA_ERR_WORKSPACE;
  return run(a, false);
}

int fla_sm100_recurrence_bwd(const FlaRecurrenceArgs* a) {
  if (const int rc = check(a)) return rc;
  if (a->d_x.ptr == nullptr && a->d_g.ptr == nullptr && a->r_final == nullptr) return FLA_ERR_INVALID;
  if (a->states == nullptr || a->states_bytes < fla_sm100_recurrence_states_bytes(a)) return FLA_ERR_WORKSPACE;
  return run(a, true);
}

}  // extern "C"
