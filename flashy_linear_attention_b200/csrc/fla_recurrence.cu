// Gated linear recurrence for sm_100a: every channel of a head carries a state of its own,
//     h_t = exp(g_t) h_(t-1) + x_t,      out_t = h_t,
// and with G_t = dO_t + R_(t+1), R_t = exp(g_t) G_t the gradients are
//     dx_t = G_t,   dg_t = R_t h_(t-1),  d(s_init) = R_0,  R_N = d(s_final).
// The reference has no counterpart (its mixers are products of q, k and v, flashlinear/linear_attn.py:11-31).
//
// Bound by HBM: two multiply-adds and an exp an element next to 6 bytes (16-bit rows; the backward 10). What it
// takes is that enough of a sequence is in flight although each token waits for the one before. A token is a map
// c -> a c + b, and the composition of such maps is one again, so a run of T tokens is summed from zero
// (b) with its decay (a = exp of the sum of its g) without knowing what came before:
//   * a thread has two channels of a run of T = 16 tokens (8 where rows or gates are fp32);
//   * the runs of a CTA exchange (a, b) through shared memory, the CTAs of a cluster, which share a tile of channels
//     and take neighbouring stretches of tokens, through distributed shared memory, both in one fixed order;
//   * then each run is walked again from the state before it.
// A cluster walks its sequence from end to end, the rows of the next steps being on their way while it
// exchanges. Nothing is read from memory twice, there is no scratch and no atomic on data, and the order of all sums
// depends on shapes and strides only. For the backward the forward keeps the state before every run (fp32, 4 and 2.5 % more
// traffic of the two passes with 16-bit rows), from which the states inside are formed again.
//
// Four ways, by what rows allow: short sequences alone in a warp; rows on 16-byte or 4-byte boundaries through tiles in
// shared memory; 16-bit rows of odd widths by direct loads. Measured (B200, of the 6.45 TB/s of a copy): 4 x 32 heads,
// 8192 x 128 in bf16 forward 146 us (85 %), backward 236 (88 %), a tenth more once the GPU draws its full power; 65536 tokens of
// 8 x 128 channels with fp32 gates 152 (55 %) and 270 (54 %); 3 x 24 heads, 1984 x 83 in fp32 74 (30 %) and 88 (42 %): the 4-byte
// copies; 4 x 32 heads, 8192 x 83 in bf16 299 (27 %) and 580 (23 %): direct loads of single elements, whose registers spill. Few
// channels are bound by the time of a step (1.2 us, 2 in a cluster of eight), whatever the rows hold: 65536 tokens of
// 64 channels 68 and 127 us.
//
// Accuracy. Channels with a memory of ten thousand tokens multiply the state by exp(-1e-4) as often. That
// factor rounded to 32 bits is off by up to 3e-8, every time in the same direction. The state is therefore multiplied
// once a run, by exp(sum of g) held as two floats; the decays of single tokens only act within a run. 16-bit rows take those from the
// fast exponential (off by 2^-22), which is all that their fp32 results (states, and gradients of fp32 gates) are off by beyond roundings.
//
// A gate of minus infinity (a document starts) drops the state whatever it holds, infinities and NaN included, whatever gates stand
// beside it, and nothing flows back past it.
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
  int* status;
  unsigned long long wait_limit_ns;
  int withhold;               // the first map of rank 0 is never sent (a test of the wait's limit)
  int tiles;                  // tiles of channels a (batch, head)
  long long tiles_all;
};

constexpr int kShortThreads = 128;
constexpr int kRecMaxCluster = 8;  // (what the exchange holds in registers)

// Tokens of a run: what a thread has registers for.
template <typename TX, typename TG>
constexpr int kRunTokens = sizeof(TX) + sizeof(TG) <= 4 ? 16 : 8;

// The map of a run, c -> (hi + lo) c + b, for two channels. hi < 0: the run drops what came before.
struct RunMap {
  float2 hi, lo, b;
};

// A factor that underflows leaves nothing of a state, however large, but an infinity stays one until a gate of minus infinity (and
// without `lo`, which would make a NaN of two opposite ones).
constexpr float kLeastDecay = 1.17549435e-38f, kMostDecay = 3.40282347e38f;
__device__ __forceinline__ float apply_map(float c, float hi, float lo, float b) {
  const float finite = fmaf(hi, c, fmaf(lo, c, b)), infinite = fmaf(hi < kLeastDecay ? kLeastDecay : hi, c, b);
  return hi < 0.f ? b : fabsf(c) <= kMostDecay ? finite : infinite;
}
__device__ __forceinline__ float2 apply_map(float2 c, const RunMap& m) {
  return make_float2(apply_map(c.x, m.hi.x, m.lo.x, m.b.x), apply_map(c.y, m.hi.y, m.lo.y, m.b.y));
}

// 2^x, off by 2^-22 of it; results below the normal numbers are zero.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.44269504f;

// exp(s) as hi + lo. Near 1, where the error of one float would act on a long memory, the second takes up what the
// first lost: exp(s) - 1 from its series (s^7 / 5040 is below 2^-31 of it there). Further off the memory ends within
// eight runs, and the fast exponential will do.
__device__ __forceinline__ void split_exp(float s, float* hi, float* lo) {
  float e = fmaf(s, 1.f / 720.f, 1.f / 120.f);
  e = fmaf(s, e, 1.f / 24.f);
  e = fmaf(s, e, 1.f / 6.f);
  e = fmaf(s, e, 0.5f);
  e = fmaf(s * s, e, s);
  const bool near = fabsf(s) < 0.125f;
  *hi = near ? 1.f + e : s == -INFINITY ? -1.f : fast_exp2(s * kLog2e);
  *lo = near ? e - (*hi - 1.f) : 0.f;
}
__device__ __forceinline__ RunMap token_map(float2 g, float2 b) {
  RunMap m;
  m.b = b;
  split_exp(g.x, &m.hi.x, &m.lo.x);
  split_exp(g.y, &m.hi.y, &m.lo.y);
  return m;
}
// (a run's factor past the largest number leaves a state of zero zero)
__device__ __forceinline__ float at_most(float hi) { return hi > kMostDecay ? kMostDecay : hi; }
__device__ __forceinline__ RunMap run_map(float2 sum, float2 b) {
  RunMap m = token_map(sum, b);
  m.hi = make_float2(at_most(m.hi.x), at_most(m.hi.y));
  return m;
}

// Decays of one token. 16-bit rows: the fast exponential, whose error acts on the tokens of a run only.
template <typename TX>
__device__ __forceinline__ float2 decay(float2 g) {
  if (sizeof(TX) == 4) return make_float2(expf(g.x), expf(g.y));
  const float2 e = mul2(g, make_float2(kLog2e, kLog2e));
  return make_float2(fast_exp2(e.x), fast_exp2(e.y));
}
// DROPS: some gate of the run is minus infinity; the state before it goes even if it is not finite.
template <typename TX, bool DROPS>
__device__ __forceinline__ float2 advance(float2 g, float2 h, float2 x) {
  float2 r = fma2(decay<TX>(g), h, x);
  if (DROPS) {
    if (g.x == -INFINITY) r.x = x.x;
    if (g.y == -INFINITY) r.y = x.y;
  }
  return r;
}
// The same step backward, R_t = exp(g) G_t. The backward kernels carry G and not R from token to token, G_t = dO_t +
// exp(g_(t+1)) G_(t+1) in one operation wherever it is formed: as a product and a sum it is compiled to one in some of the walks
// and to two in others, and the bits of a channel then depend on whether another one's gates call for a careful walk.
template <typename TX, bool DROPS>
__device__ __forceinline__ float2 retreat(float2 g, float2 all) {
  float2 r = mul2(decay<TX>(g), all);
  if (DROPS) {
    if (g.x == -INFINITY) r.x = 0.f;
    if (g.y == -INFINITY) r.y = 0.f;
  }
  return r;
}

// Whether a run drops the state is read from the sum of its gates, which is minus infinity then, unless a NaN or plus infinity
// among them made it NaN: a run with such a sum is looked through (mark_drops), and its sum is minus infinity again from there on.
__device__ __forceinline__ bool may_drop(float2 sum) { return !(sum.x > -INFINITY && sum.y > -INFINITY); }
__device__ __forceinline__ bool no_number(float2 sum) { return sum.x != sum.x || sum.y != sum.y; }
__device__ __forceinline__ void mark_drops(float2 gate, float2* sum) {
  if (gate.x == -INFINITY) sum->x = -INFINITY;
  if (gate.y == -INFINITY) sum->y = -INFINITY;
}

struct Place {  // what a thread works on
  int b, h, c0, gap;
  bool ok0, ok1;
};
template <bool PAIR, int LPR>
__device__ __forceinline__ Place place(const RecurrenceParams& p, long long tile, int lane) {
  Place w;
  const long long bh = tile / p.tiles;
  w.b = static_cast<int>(bh / p.heads);
  w.h = static_cast<int>(bh % p.heads);
  w.gap = PAIR ? 1 : LPR;
  w.c0 = static_cast<int>(tile % p.tiles) * 2 * LPR + (PAIR ? 2 * lane : lane);
  w.ok0 = w.c0 < p.c;
  w.ok1 = w.c0 + w.gap < p.c;
  return w;
}
// Index into RecurrenceParams::states, whose layout does not depend on how heads were joined.
__device__ __forceinline__ long long state_of(const RecurrenceParams& p, const Place& w, int run, int runs_all) {
  return ((static_cast<long long>(w.b) * runs_all + run) * p.heads + w.h) * p.c + w.c0;
}

// ------------------------------------------------------------------------------------------------------------
// Short sequences, and rows so far apart that their offsets need 64 bits: every group of LPR lanes walks a tile of
// channels alone, token by token. A program that decodes multiplies its state once a call by one token's decay, so
// that is split in two floats here.

template <typename T>
__device__ __forceinline__ T* row0(const RecurrenceTensor& t, const Place& w) {
  return static_cast<T*>(t.ptr) + w.b * t.sb + w.h * t.sh + w.c0;
}

template <typename TX, typename TG, bool PAIR, int LPR>
__global__ void __launch_bounds__(kShortThreads) fla_recurrence_short_fwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  const long long tile = static_cast<long long>(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  if (tile >= p.tiles_all) return;
  const Place w = place<PAIR, LPR>(p, tile, threadIdx.x % LPR);
  const TX* xp = row0<const TX>(p.x, w);
  const TG* gp = row0<const TG>(p.g, w);
  TX* op = row0<TX>(p.o, w);
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  const int runs_all = (p.n - 1) / T + 1;
  float2 h = make_float2(0.f, 0.f);
  if (p.start != nullptr) h = load_pair<float, PAIR>(p.start + cell, w.gap, w.ok0, w.ok1);
  for (int run = 0; run < runs_all; ++run) {
    const int t0 = run * T;
    if (p.states != nullptr) store_pair<float, PAIR>(p.states + state_of(p, w, run, runs_all), w.gap, w.ok0, w.ok1, h);
    typename PairOf<TX>::Raw x[T];
    typename PairOf<TG>::Raw g[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const bool in = t0 + t < p.n;
      x[t] = load_pair<TX, PAIR>(xp + (t0 + t) * p.x.sn, w.gap, w.ok0 && in, w.ok1 && in);
      g[t] = load_pair<TG, PAIR>(gp + (t0 + t) * p.g.sn, w.gap, w.ok0 && in, w.ok1 && in);
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (t0 + t >= p.n) break;
      h = apply_map(h, token_map(unpack_pair<TG>(g[t]), unpack_pair<TX>(x[t])));
      store_pair<TX, PAIR>(op + (t0 + t) * p.o.sn, w.gap, w.ok0, w.ok1, h);
    }
  }
  if (p.end != nullptr) store_pair<float, PAIR>(p.end + cell, w.gap, w.ok0, w.ok1, h);
}

template <typename TX, typename TG, bool PAIR, int LPR>
__global__ void __launch_bounds__(kShortThreads) fla_recurrence_short_bwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  const long long tile = static_cast<long long>(blockIdx.x) * (kShortThreads / LPR) + threadIdx.x / LPR;
  if (tile >= p.tiles_all) return;
  const Place w = place<PAIR, LPR>(p, tile, threadIdx.x % LPR);
  const TX* xp = row0<const TX>(p.x, w);
  const TG* gp = row0<const TG>(p.g, w);
  const TX* yp = row0<const TX>(p.o, w);
  TX* dxp = row0<TX>(p.dx, w);
  TG* dgp = row0<TG>(p.dg, w);
  const bool has_dy = p.o.ptr != nullptr;
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  const int runs_all = (p.n - 1) / T + 1;
  float2 r = make_float2(0.f, 0.f);
  if (p.start != nullptr) r = load_pair<float, PAIR>(p.start + cell, w.gap, w.ok0, w.ok1);
  for (int run = runs_all - 1; run >= 0; --run) {
    const int t0 = run * T;
    typename PairOf<TX>::Raw x[T], y[T];
    typename PairOf<TG>::Raw g[T];
    float2 h = load_pair<float, PAIR>(p.states + state_of(p, w, run, runs_all), w.gap, w.ok0, w.ok1);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const bool in = t0 + t < p.n;
      x[t] = load_pair<TX, PAIR>(xp + (t0 + t) * p.x.sn, w.gap, w.ok0 && in, w.ok1 && in);
      g[t] = load_pair<TG, PAIR>(gp + (t0 + t) * p.g.sn, w.gap, w.ok0 && in, w.ok1 && in);
      y[t] = load_pair<TX, PAIR>(yp + (t0 + t) * p.o.sn, w.gap, w.ok0 && in && has_dy, w.ok1 && in && has_dy);
    }
    float2 before[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      before[t] = h;
      h = apply_map(h, token_map(unpack_pair<TG>(g[t]), unpack_pair<TX>(x[t])));
    }
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      if (t0 + t >= p.n) continue;
      const float2 gv = unpack_pair<TG>(g[t]), all = add2(unpack_pair<TX>(y[t]), r);
      if (p.dx.ptr != nullptr) store_pair<TX, PAIR>(dxp + (t0 + t) * p.dx.sn, w.gap, w.ok0, w.ok1, all);
      r = apply_map(all, token_map(gv, make_float2(0.f, 0.f)));
      if (p.dg.ptr != nullptr)
        store_pair<TG, PAIR>(dgp + (t0 + t) * p.dg.sn, w.gap, w.ok0, w.ok1,
                             make_float2(gv.x == -INFINITY ? 0.f : r.x * before[t].x, gv.y == -INFINITY ? 0.f : r.y * before[t].y));
    }
  }
  if (p.end != nullptr) store_pair<float, PAIR>(p.end + cell, w.gap, w.ok0, w.ok1, r);
}

// ------------------------------------------------------------------------------------------------------------
// Clusters of CTAs that walk a tile of 2 LPR channels together, a step of ranks * runs * T tokens at a time.

// What the threads of a CTA, and the CTAs of a cluster, hand each other of a step.
struct JoinSpace {
  RunMap* run;      // [run of the CTA][lane]
  float2* before;   // the same: a run's sum of gates, and then the state before it
  float4* factor;   // [step parity][rank][lane]: hi and lo of the CTAs' maps
  float2* b;        // the same
  uint64_t* arrived;  // [step parity]: barriers
};
template <int LPR, int THREADS>
struct RecurrenceShared {
  RunMap run[THREADS];
  float2 before[THREADS];
  float4 factor[2 * kRecMaxCluster * LPR];
  float2 b[2 * kRecMaxCluster * LPR];
  uint64_t arrived[2];
  __device__ __forceinline__ JoinSpace space() { return {run, before, factor, b, arrived}; }
};
struct Team {
  int lane, run, rank, ranks;
};

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t peer_address(uint32_t address, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}

// Waits until the maps of all peers have arrived; false if that takes longer than the limit.
__device__ __forceinline__ bool maps_arrived(uint32_t barrier, uint32_t phase, unsigned long long limit_ns) {
  unsigned long long start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(barrier), "r"(phase)
        : "memory");
    if (done) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - start > limit_ns) return false;
  }
}

// Sends this CTA's map of a step to every CTA of the cluster, itself included, and waits for theirs. The stores count
// their bytes at the receiver's barrier when they have arrived: unlike a barrier of the cluster, they need no fence, and
// so do not wait for the rows that were written to memory before (65536 tokens of 64 channels: 348 us that way, 150 this
// way, with 512 tokens a step). A peer
// writes to a slot again two steps later, for which it needs what this CTA sends when it has read the slot.
template <int LPR>
__device__ __forceinline__ bool trade_maps(const JoinSpace& sh, int step, const RunMap& all, const Team& w,
                                           const RecurrenceParams& p) {
  const int parity = step & 1;
  const uint32_t factor = shared_address(sh.factor + (parity * kRecMaxCluster + w.rank) * LPR + w.lane);
  const uint32_t b = shared_address(sh.b + (parity * kRecMaxCluster + w.rank) * LPR + w.lane);
  const uint32_t barrier = shared_address(sh.arrived + parity);
  if (w.lane == 0)
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier), "r"(w.ranks * LPR * 24) : "memory");
  if (!(p.withhold && step == 0 && w.rank == 0)) {
    for (int r = 0; r < w.ranks; ++r) {
      const uint32_t bar = peer_address(barrier, r);
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                       peer_address(factor, r)),
                   "f"(all.hi.x), "f"(all.hi.y), "f"(all.lo.x), "f"(all.lo.y), "r"(bar)
                   : "memory");
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(peer_address(b, r)),
                   "f"(all.b.x), "f"(all.b.y), "r"(bar)
                   : "memory");
    }
  }
  return maps_arrived(barrier, (step >> 1) & 1, p.wait_limit_ns);
}

// Joins the maps of the runs of a step, in their order: the state before each run goes to `before`. `carry` is the state
// before the step and becomes the one behind it. Runs and ranks count in the direction of the walk. One thread a pair of
// channels does it (all warps doing so for themselves issued a tenth of the kernel's instructions). `lost`: a wait has run
// out; the state is NaN from there on, and nothing is sent or waited for any more.
template <int LPR, int RUNS>
__device__ __forceinline__ void join(const JoinSpace& sh, int step, const Team& w, const RecurrenceParams& p, float2& carry, bool& lost) {
  // (eight maps at a time in registers: loads between the steps of the chain cost 100 cycles a run)
  constexpr int kSome = 8;
  static_assert(RUNS % kSome == 0 && kRecMaxCluster == kSome, "");
  RunMap m[kSome];
  auto some = [&](int from) {
#pragma unroll
    for (int i = 0; i < kSome; ++i) m[i] = sh.run[(from + i) * LPR + w.lane];
  };
  float2 c = carry;
  if (w.ranks > 1) {
    float2 sum = make_float2(0.f, 0.f), b = sum;
#pragma unroll
    for (int from = 0; from < RUNS; from += kSome) {
      float2 sums[kSome];
#pragma unroll
      for (int i = 0; i < kSome; ++i) sums[i] = sh.before[(from + i) * LPR + w.lane];
      some(from);
#pragma unroll
      for (int i = 0; i < kSome; ++i) {
        sum = add2(sum, sums[i]);
        b = apply_map(b, m[i]);
      }
    }
    if (no_number(sum)) {  // (one run's NaN hides that another drops)
#pragma unroll 1
      for (int i = 0; i < RUNS; ++i) {
        const float2 hi = sh.run[i * LPR + w.lane].hi;
        mark_drops(make_float2(hi.x < 0.f ? -INFINITY : 0.f, hi.y < 0.f ? -INFINITY : 0.f), &sum);
      }
    }
    if (!lost && !trade_maps<LPR>(sh, step, run_map(sum, b), w, p)) {
      lost = true;
      if (p.status != nullptr) atomicOr(p.status, 1);
    }
#pragma unroll
    for (int r = 0; r < kRecMaxCluster; ++r) {
      const int at = ((step & 1) * kRecMaxCluster + (r < w.ranks ? r : 0)) * LPR + w.lane;
      const float4 f = sh.factor[at];
      m[r].hi = make_float2(f.x, f.y);
      m[r].lo = make_float2(f.z, f.w);
      m[r].b = sh.b[at];
    }
    float2 before = c;
#pragma unroll
    for (int r = 0; r < kRecMaxCluster; ++r)
      if (r < w.ranks) {
        if (r == w.rank) before = c;
        c = apply_map(c, m[r]);
      }
    if (lost) c = before = make_float2(NAN, NAN);
    carry = c;
    c = before;
  }
#pragma unroll
  for (int from = 0; from < RUNS; from += kSome) {
    some(from);
#pragma unroll
    for (int i = 0; i < kSome; ++i) {
      sh.before[(from + i) * LPR + w.lane] = c;
      c = apply_map(c, m[i]);
    }
  }
  if (w.ranks == 1) carry = c;
}

// The exchange of a step by the threads that work on it: the first run's join, the others wait for them.
template <int LPR, int THREADS>
__device__ __forceinline__ float2 exchange(RecurrenceShared<LPR, THREADS>& sh, int step, float2 sum, float2 b, const Team& w,
                                           const RecurrenceParams& p, float2& carry, bool& lost) {
  sh.run[w.run * LPR + w.lane] = run_map(sum, b);
  sh.before[w.run * LPR + w.lane] = sum;
  __syncthreads();
  if (w.run == 0) join<LPR, THREADS / LPR>(sh.space(), step, w, p, carry, lost);
  __syncthreads();
  return sh.before[w.run * LPR + w.lane];
}

template <bool PAIR, int LPR>
__device__ __forceinline__ void take_place(const RecurrenceParams& p, uint64_t* arrived, Team* team, Place* w) {
  cg::cluster_group cluster = cg::this_cluster();
  team->lane = threadIdx.x % LPR;
  team->run = threadIdx.x / LPR;
  team->ranks = cluster.num_blocks();
  team->rank = cluster.block_rank();
  *w = place<PAIR, LPR>(p, blockIdx.x / team->ranks, team->lane);
  if (threadIdx.x == 0 && team->ranks > 1) {
    for (int i = 0; i < 2; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(arrived + i)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
}

// Keeps the compiler from carrying what it derived from a value (decays, offsets) from one loop to the next: it has them
// all in registers then, and those in memory.
__device__ __forceinline__ void anew(uint32_t& v) { asm volatile("" : "+r"(v)); }
__device__ __forceinline__ void anew(float2& v) { asm volatile("" : "+f"(v.x), "+f"(v.y)); }
template <typename R, int T>
__device__ __forceinline__ void anew(R (&v)[T]) {
#pragma unroll
  for (int t = 0; t < T; ++t) anew(v[t]);
}

__device__ __forceinline__ void load_after(uint16_t& r, const char* q, float after) {
  asm volatile("ld.global.nc.b16 %0, [%1];" : "=h"(r) : "l"(q), "f"(after));
}
__device__ __forceinline__ void load_after(float& r, const char* q, float after) {
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(r) : "l"(q), "f"(after));
}

// A thread's two columns of the rows of a step: the rows' base is the same for the CTA, offsets inside a step fit 32 bits
// (checked on the host). Columns past the last read the first one's and are not written.
template <typename T>
struct Rows {
  char* base;  // of the batch entry and head
  uint32_t at, gap, row;  // bytes

  __device__ __forceinline__ Rows(const RecurrenceTensor& t, const Place& w, int first) {
    base = static_cast<char*>(t.ptr) + (w.b * t.sb + w.h * t.sh) * static_cast<long long>(sizeof(T));
    row = static_cast<uint32_t>(t.sn) * sizeof(T);
    at = (w.ok0 ? w.c0 * sizeof(T) : 0u) + first * row;
    gap = w.ok1 ? w.gap * sizeof(T) : 0u;
  }
  __device__ __forceinline__ char* step(const RecurrenceTensor& t, long long token) const {
    return base + token * t.sn * static_cast<long long>(sizeof(T));
  }
  // `after`: the load is issued behind what this value comes from, whose operands' registers it can take.
  __device__ __forceinline__ typename PairOf<T>::Raw load(const char* step, uint32_t token, float after) const {
    const char* q = step + (at + token * row);
    typename PairOf<T>::Element a, b;
    load_after(a, q, after);
    load_after(b, q + gap, after);
    return join_pair(a, b);
  }
  __device__ __forceinline__ void store(char* step, uint32_t token, const Place& w, float2 v) const {
    store_pair<T, false>(reinterpret_cast<T*>(step + (at + token * row)), w.gap, w.ok0, w.ok1, v);
  }
};

// Runs with a gate of minus infinity, of which there are few, are summed out of line and from memory: in line their
// second copy of the loops cost the kernels 50 registers.
template <typename TX, typename TG, int T>
__device__ __noinline__ float2 advance_from(float2 h, const typename PairOf<TX>::Raw* x, const typename PairOf<TG>::Raw* g,
                                            float2* before) {
#pragma unroll 1
  for (int t = 0; t < T; ++t) {
    if (before != nullptr) before[t] = h;
    h = advance<TX, true>(unpack_pair<TG>(g[t]), h, unpack_pair<TX>(x[t]));
  }
  return h;
}
// R before a run from zero behind it, with what a gate of minus infinity drops left out.
template <typename TX, typename TG, int T>
__device__ __noinline__ float2 retreat_from_zero(const typename PairOf<TX>::Raw* y, const typename PairOf<TG>::Raw* g) {
  float2 all = make_float2(0.f, 0.f), gate = all;  // gate: the one behind the token
#pragma unroll 1
  for (int t = T - 1; t >= 0; --t) {
    const float2 yv = unpack_pair<TX>(y[t]);
    all = t == T - 1 ? yv : advance<TX, true>(gate, all, yv);
    gate = unpack_pair<TG>(g[t]);
  }
  return retreat<TX, true>(gate, all);
}
template <typename TG, int T>
__device__ __noinline__ float2 sum_with_drops(float2 sum, const typename PairOf<TG>::Raw* g) {
#pragma unroll 1
  for (int t = 0; t < T; ++t) mark_drops(unpack_pair<TG>(g[t]), &sum);
  return sum;
}
template <typename R, int T>
struct InMemory {
  R v[T];
  __device__ __forceinline__ explicit InMemory(const R (&from)[T]) {
#pragma unroll
    for (int t = 0; t < T; ++t) v[t] = from[t];
  }
};

template <typename TX, typename TG, int LPR, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) fla_recurrence_direct_fwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  __shared__ RecurrenceShared<LPR, THREADS> sh;
  Team team;
  Place w;
  take_place<false, LPR>(p, sh.arrived, &team, &w);
  bool lost = false;
  const int first = (team.rank * (THREADS / LPR) + team.run) * T;  // of the step's tokens
  Rows<TX> xr(p.x, w, first), orow(p.o, w, first);
  Rows<TG> gr(p.g, w, first);
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  if (team.run == 0 && p.start != nullptr) carry = load_pair<float, false>(p.start + cell, w.gap, w.ok0, w.ok1);

  const int span = team.ranks * (THREADS / LPR) * T;  // tokens a step
  const int steps = (p.n - 1) / span + 1, runs_all = (p.n - 1) / T + 1;
  typename PairOf<TX>::Raw x[T];
  typename PairOf<TG>::Raw g[T];
  auto fetch = [&](int t, int step, float after) {  // one token of the step; none behind the last: the identity
    zero_pair(x[t]);
    zero_pair(g[t]);
    if (step * span + first + t < p.n) {
      x[t] = xr.load(xr.step(p.x, static_cast<long long>(step) * span), t, after);
      g[t] = gr.load(gr.step(p.g, static_cast<long long>(step) * span), t, after);
    }
  };
#pragma unroll
  for (int t = 0; t < T; ++t) fetch(t, 0, 0.f);
  if (team.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
  for (int step = 0; step < steps; ++step) {
    const int t0 = step * span + first;
    float2 sum = make_float2(0.f, 0.f), h = sum;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float2 gv = unpack_pair<TG>(g[t]);
      sum = add2(sum, gv);
      h = advance<TX, false>(gv, h, unpack_pair<TX>(x[t]));
    }
    const bool drops = __any_sync(0xffffffffu, may_drop(sum));
    if (drops) {
      const InMemory<typename PairOf<TX>::Raw, T> xm(x);
      const InMemory<typename PairOf<TG>::Raw, T> gm(g);
      if (__any_sync(0xffffffffu, no_number(sum))) sum = sum_with_drops<TG, T>(sum, gm.v);
      h = advance_from<TX, TG, T>(make_float2(0.f, 0.f), xm.v, gm.v, nullptr);
    }
    h = exchange(sh, step, sum, h, team, p, carry, lost);
    if (p.states != nullptr && t0 < p.n)
      store_pair<float, false>(p.states + state_of(p, w, t0 / T, runs_all), w.gap, w.ok0, w.ok1, h);
    char* os = orow.step(p.o, static_cast<long long>(step) * span);
    anew(x);
    anew(g);
    anew(xr.row);
    anew(gr.row);
    anew(orow.row);
    if (!drops && (step + 2) * span <= p.n) {  // this step and the next are whole
      const char* xs = xr.step(p.x, static_cast<long long>(step + 1) * span);
      const char* gs = gr.step(p.g, static_cast<long long>(step + 1) * span);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        h = advance<TX, false>(unpack_pair<TG>(g[t]), h, unpack_pair<TX>(x[t]));
        orow.store(os, t, w, h);
        x[t] = xr.load(xs, t, h.x);  // the next step's, as soon as its place is free
        g[t] = gr.load(gs, t, h.x);
      }
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        h = advance<TX, true>(unpack_pair<TG>(g[t]), h, unpack_pair<TX>(x[t]));
        if (t0 + t < p.n) orow.store(os, t, w, h);
        fetch(t, step + 1, h.x);
      }
    }
  }
  if (p.end != nullptr && team.run == 0 && team.rank == 0)
    store_pair<float, false>(p.end + cell, w.gap, w.ok0, w.ok1, carry);
  if (team.ranks > 1) cg::this_cluster().sync();  // (nobody leaves while a peer that gave up early may still be written to)
}

template <typename TX, typename TG, int LPR, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) fla_recurrence_direct_bwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>;
  __shared__ RecurrenceShared<LPR, THREADS> sh;
  Team team;
  Place w;
  take_place<false, LPR>(p, sh.arrived, &team, &w);
  bool lost = false;
  const int span = team.ranks * (THREADS / LPR);                        // runs a step
  const int nth = span - 1 - (team.rank * (THREADS / LPR) + team.run);  // of the step's runs, in the order of the tokens
  const int first = nth * T;
  Rows<TX> xr(p.x, w, first), yr(p.o, w, first), dxr(p.dx, w, first);
  Rows<TG> gr(p.g, w, first), dgr(p.dg, w, first);
  const bool has_dy = p.o.ptr != nullptr, want_dx = p.dx.ptr != nullptr, want_dg = p.dg.ptr != nullptr;
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  if (team.run == 0 && p.start != nullptr) carry = load_pair<float, false>(p.start + cell, w.gap, w.ok0, w.ok1);

  const int runs_all = (p.n - 1) / T + 1;
  const int steps = (runs_all - 1) / span + 1;
  typename PairOf<TX>::Raw x[T], y[T];
  typename PairOf<TG>::Raw g[T];
  float2 state;
  auto rows_x = [&](int t, int step, float after) {
    zero_pair(x[t]);
    if (step * span * T + first + t < p.n) x[t] = xr.load(xr.step(p.x, static_cast<long long>(step) * span * T), t, after);
  };
  auto rows_gy = [&](int t, int step, float after) {
    zero_pair(g[t]);
    zero_pair(y[t]);
    if (step * span * T + first + t < p.n) {
      g[t] = gr.load(gr.step(p.g, static_cast<long long>(step) * span * T), t, after);
      if (has_dy) y[t] = yr.load(yr.step(p.o, static_cast<long long>(step) * span * T), t, after);
    }
  };
  auto load_state = [&](int step) {
    state = make_float2(0.f, 0.f);
    const int run = step * span + nth;
    if (run < runs_all) state = load_pair<float, false>(p.states + state_of(p, w, run, runs_all), w.gap, w.ok0, w.ok1);
  };
  load_state(steps - 1);
#pragma unroll
  for (int t = 0; t < T; ++t) rows_x(t, steps - 1, 0.f);
#pragma unroll
  for (int t = T - 1; t >= 0; --t) rows_gy(t, steps - 1, 0.f);
  if (team.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
  // The walk starts at the end; the runs behind the last token are the identity. Steps before the last one are whole.
  for (int step = steps - 1; step >= 0; --step) {
    float2 sum = make_float2(0.f, 0.f), r = sum, a = sum, h = state;
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      const float2 gv = unpack_pair<TG>(g[t]);
      sum = add2(sum, gv);
      r = t == T - 1 ? unpack_pair<TX>(y[t]) : fma2(a, r, unpack_pair<TX>(y[t]));
      a = decay<TX>(gv);
    }
    r = mul2(a, r);
    const bool drops = __any_sync(0xffffffffu, may_drop(sum));
    float2 before[T];  // the state before each token
    anew(g);
    if (drops) {
      const InMemory<typename PairOf<TX>::Raw, T> xm(x), ym(y);
      const InMemory<typename PairOf<TG>::Raw, T> gm(g);
      float2 bm[T];
      if (__any_sync(0xffffffffu, no_number(sum))) sum = sum_with_drops<TG, T>(sum, gm.v);
      r = retreat_from_zero<TX, TG, T>(ym.v, gm.v);
      advance_from<TX, TG, T>(h, xm.v, gm.v, bm);
#pragma unroll
      for (int t = 0; t < T; ++t) before[t] = bm[t];
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        before[t] = h;
        h = advance<TX, false>(unpack_pair<TG>(g[t]), h, unpack_pair<TX>(x[t]));
      }
    }
    anew(y);
    anew(g);
    anew(xr.row);
    if (step > 0) {  // x and the state are done with: the next step's
      load_state(step - 1);
      const char* xs = xr.step(p.x, static_cast<long long>(step - 1) * span * T);
#pragma unroll
      for (int t = 0; t < T; ++t) x[t] = xr.load(xs, t, before[t].x);
    }
    r = exchange(sh, steps - 1 - step, sum, r, team, p, carry, lost);
    const long long token = static_cast<long long>(step) * span * T;
    anew(yr.row);
    anew(gr.row);
    anew(dxr.row);
    anew(dgr.row);
    char *dxs = dxr.step(p.dx, token), *dgs = dgr.step(p.dg, token);
    if (!drops && step > 0 && step < steps - 1 && has_dy && want_dx && want_dg) {
      const char *ys = yr.step(p.o, token - static_cast<long long>(span) * T), *gs = gr.step(p.g, token - static_cast<long long>(span) * T);
#pragma unroll
      for (int t = T - 1; t >= 0; --t) {
        const float2 all = t == T - 1 ? add2(unpack_pair<TX>(y[t]), r) : fma2(a, r, unpack_pair<TX>(y[t]));
        dxr.store(dxs, t, w, all);
        a = decay<TX>(unpack_pair<TG>(g[t]));
        dgr.store(dgs, t, w, mul2(mul2(a, all), before[t]));
        r = all;
        y[t] = yr.load(ys, t, r.x);
        g[t] = gr.load(gs, t, r.x);
      }
    } else {
      float2 gate = make_float2(0.f, 0.f);  // the one behind the token
#pragma unroll
      for (int t = T - 1; t >= 0; --t) {
        const float2 gv = unpack_pair<TG>(g[t]), yv = unpack_pair<TX>(y[t]);
        const float2 all = t == T - 1 ? add2(yv, r) : advance<TX, true>(gate, r, yv);
        const bool in = token + first + t < p.n;
        if (in && want_dx) dxr.store(dxs, t, w, all);
        r = all;
        gate = gv;
        if (in && want_dg) {
          float2 d = mul2(mul2(decay<TX>(gv), all), before[t]);
          if (gv.x == -INFINITY) d.x = 0.f;
          if (gv.y == -INFINITY) d.y = 0.f;
          dgr.store(dgs, t, w, d);
        }
        if (step > 0) rows_gy(t, step - 1, r.x);
      }
    }
  }
  if (p.end != nullptr && team.run == 0 && team.rank == 0)
    store_pair<float, false>(p.end + cell, w.gap, w.ok0, w.ok1, carry);
  if (team.ranks > 1) cg::this_cluster().sync();  // (nobody leaves while a peer that gave up early may still be written to)
}

// ------------------------------------------------------------------------------------------------------------
// The same with rows that lie on 4-byte boundaries, or better on 16: a warp brings the rows of its runs of the next steps into
// a tile of its own in shared memory, asynchronously, and lets results leave the same way. The loads of a step so are on
// their way through the whole step before, its exchange included, and with 16 bytes a lane there are a quarter as many.

// T-typed rows of the runs of a warp: TOK tokens each, 2 LPR columns, copied in pieces of PIECE bytes: 16, or 4 where
// rows are aligned to no more.
template <typename T, int LPR, int TOK, int PIECE>
struct WarpTile {
  static constexpr int kRow = 2 * LPR * sizeof(T), kPieces = kRow / PIECE, kRows = TOK * (32 / LPR);
  static constexpr int kBytes = kRows * kRow, kEach = kBytes / (32 * PIECE);
  static constexpr int kRowsEach = kPieces < 32 ? 32 / kPieces : 1, kParts = kPieces > 32 ? kPieces / 32 : 1;  // a row a turn, or parts of it
  char* base;                     // of the batch entry, head and tile of channels
  uint32_t at, row;               // bytes
  int first, left_in_row;         // the lane's first row of the warp's; bytes of the row from its piece on
  bool whole;                     // every piece lies inside the row

  __device__ __forceinline__ WarpTile(const RecurrenceTensor& t, const Place& w, int tile_column, int columns, int first_token) {
    base = static_cast<char*>(t.ptr) + (w.b * t.sb + w.h * t.sh + tile_column) * static_cast<long long>(sizeof(T));
    row = static_cast<uint32_t>(t.sn) * sizeof(T);
    const int lane = threadIdx.x % 32, piece = lane % kPieces;
    first = lane / kPieces;
    at = (first_token + first) * row + piece * PIECE;
    left_in_row = columns * static_cast<int>(sizeof(T)) - piece * PIECE;
    whole = columns >= 2 * LPR;
  }
  __device__ __forceinline__ char* step(const RecurrenceTensor& t, long long token) const {
    return base + token * t.sn * static_cast<long long>(sizeof(T));
  }
  __device__ __forceinline__ bool inside(int k, int left) const {
    return k % kParts * 32 * PIECE < left_in_row && first + k / kParts * kRowsEach < left;
  }
  __device__ __forceinline__ uint32_t offset(int k) const { return k / kParts * kRowsEach * row + k % kParts * 32 * PIECE; }
  // Rows past the last token (`left`: how many of the warp's rows there are) are zero, the identity.
  __device__ __forceinline__ void copy(uint32_t tile, const char* step, int left) const {
    const char* from = step + at;
    const uint32_t to = tile + threadIdx.x % 32 * PIECE;
    const bool all = left >= kRows && whole;
    if constexpr (PIECE == 16) {
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        if (all) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * 512), "l"(from + offset(k)) : "memory");
        } else {
          const bool ok = inside(k, left);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * 512), "l"(ok ? from + offset(k) : base), "r"(ok ? 16 : 0)
                       : "memory");
        }
      }
    } else {
      // (four times as many: addresses are advanced, and whole tiles make no choices, which were half of all instructions)
      const uint32_t next = kRowsEach * row;
      if (all) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + k * 128), "l"(from + k % kParts * 128) : "memory");
          if (k % kParts == kParts - 1) from += next;
        }
      } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          const bool ok = inside(k, left);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + k * 128), "l"(ok ? from + k % kParts * 128 : base), "r"(ok ? 4 : 0)
                       : "memory");
          if (k % kParts == kParts - 1) from += next;
        }
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t tile, char* step, int left) const {
    char* to = step + at;
    const bool all = left >= kRows && whole;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t from = tile + (k * 32 + threadIdx.x % 32) * PIECE;
      if constexpr (PIECE == 16) {
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
        if (all || inside(k, left)) *reinterpret_cast<uint4*>(to + offset(k)) = v;
      } else {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
        if (all || inside(k, left)) *reinterpret_cast<uint32_t*>(to + k % kParts * 128) = v;
        if (k % kParts == kParts - 1) to += kRowsEach * row;
      }
    }
  }
  // A token's two channels of a thread, whose run's rows begin at `run`.
  __device__ __forceinline__ static typename PairOf<T>::Raw get(uint32_t run, int t) {
    typename PairOf<T>::Raw r;
    if constexpr (sizeof(T) == 4)
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(run + t * kRow) : "memory");
    else
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(run + t * kRow) : "memory");
    return r;
  }
  __device__ __forceinline__ static void put(uint32_t run, int t, float2 v) {
    const auto r = pack_pair<T>(v);
    if constexpr (sizeof(T) == 4)
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(run + t * kRow), "f"(r.x), "f"(r.y) : "memory");
    else
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(run + t * kRow), "r"(r) : "memory");
  }
};
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncwarp();
}

// A gate of minus infinity needs no care as long as the state is finite: zero times it is zero. A state that is not becomes
// NaN there and stays so to the end of the run, where it is seen; only such runs are walked again with care (with selections
// in the walks themselves, or a second copy of them for every run with such a gate, packed documents of 2048 tokens cost a fifth
// of the time: 377 us without, 449 with them).
__device__ __forceinline__ bool spoilt(bool drops, float2 v) {
  return drops && __any_sync(0xffffffffu, !(fabsf(v.x) <= 3.4e38f && fabsf(v.y) <= 3.4e38f));
}

// Forward, eight warps work on runs and a ninth joins them, a step apart: while it joins the runs of one step, the others sum those
// of the next (first walk), and then finish the one before (second walk). With both on the same step (two barriers in a
// row, each waiting for a chain of one or two thousand cycles) the warps stood still for two fifths of the time.
// Three steps' tiles a warp: one that waits for its second walk, one in its first, one on its way. Results take the place
// of what they come from, and the tile is free when they have left.
constexpr int kTileThreads = 256, kTileSteps = 3;
template <int LPR>
constexpr int kJoinBytes = 2 * (kTileThreads * static_cast<int>(sizeof(RunMap) + sizeof(float2))) + 16;
template <int LPR>
constexpr int kTradeBytes = 2 * kRecMaxCluster * LPR * 24;
template <typename TX, typename TG, int LPR>
constexpr int kFwdTile = kRunTokens<TX, TG> * 64 * static_cast<int>(sizeof(TX) + sizeof(TG));
// Backward, whose tiles are larger and whose walks need more registers, two CTAs an SM with one tile a warp (and room for the
// results) each do better than one CTA a step apart: 4 x 32 heads, 8192 x 128 in bf16 235 against 336 us.
template <typename TX, typename TG, int LPR>
constexpr int kBwdTile = kRunTokens<TX, TG> * 64 * static_cast<int>(3 * sizeof(TX) + 2 * sizeof(TG));

// The joining warp's and the others' ends of the two hand-overs of a step.
enum { kMapsReady = 1, kStatesReady = 3 };  // + step parity
__device__ __forceinline__ void hand_over(int barrier) {
  asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "n"(kTileThreads + 32) : "memory");
}
__device__ __forceinline__ void take_over(int barrier) {
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kTileThreads + 32) : "memory");
}

// Shared memory: the warps' tiles, [parity] maps, [parity] sums and states, barriers, and in a cluster what is traded.
template <int LPR>
__device__ __forceinline__ JoinSpace join_space(char* after_tiles, int parity) {
  JoinSpace j;
  j.factor = reinterpret_cast<float4*>(after_tiles + kJoinBytes<LPR>);
  j.b = reinterpret_cast<float2*>(j.factor + 2 * kRecMaxCluster * LPR);
  j.run = reinterpret_cast<RunMap*>(after_tiles) + parity * kTileThreads;
  j.before = reinterpret_cast<float2*>(after_tiles + 2 * kTileThreads * sizeof(RunMap)) + parity * kTileThreads;
  j.arrived = reinterpret_cast<uint64_t*>(after_tiles + kJoinBytes<LPR> - 16);
  return j;
}
template <int LPR, int PIECE>
__device__ __forceinline__ void join_steps(const RecurrenceParams& p, char* after_tiles, Team team, const Place& w, int steps) {
  const bool active = team.lane == static_cast<int>(threadIdx.x % 32);  // (LPR = 16: half of the warp)
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  bool lost = false;
  if (p.start != nullptr) carry = load_pair<float, PIECE == 16>(p.start + cell, 1, w.ok0, w.ok1);
  for (int step = 0; step < steps; ++step) {
    take_over(kMapsReady + (step & 1));
    if (active) join<LPR, kTileThreads / LPR>(join_space<LPR>(after_tiles, step & 1), step, team, p, carry, lost);
    __syncwarp();
    hand_over(kStatesReady + (step & 1));
  }
  if (active && p.end != nullptr && team.rank == 0) store_pair<float, PIECE == 16>(p.end + cell, 1, w.ok0, w.ok1, carry);
}

template <typename TX, typename TG, int LPR, int PIECE>
__global__ void __launch_bounds__(kTileThreads + 32, 2) fla_recurrence_fwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>, kRuns = kTileThreads / LPR, kWarpRuns = 32 / LPR;
  using TileX = WarpTile<TX, LPR, T, PIECE>;
  using TileG = WarpTile<TG, LPR, T, PIECE>;
  constexpr int kTile = kFwdTile<TX, TG, LPR>;
  extern __shared__ uint4 tiles[];
  char* const after_tiles = reinterpret_cast<char*>(tiles) + kTileThreads / 32 * kTileSteps * kTile;
  Team team;
  Place w;
  take_place<true, LPR>(p, join_space<LPR>(after_tiles, 0).arrived, &team, &w);
  const int span = team.ranks * kRuns * T;  // tokens a step
  const int steps = (p.n - 1) / span + 1, runs_all = (p.n - 1) / T + 1;
  if (threadIdx.x >= kTileThreads) {
    if (team.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
    join_steps<LPR, PIECE>(p, after_tiles, team, w, steps);
  } else {
    const int column = w.c0 - 2 * team.lane;                                    // of the tile
    const int first = (team.rank * kRuns + team.run / kWarpRuns * kWarpRuns) * T;  // of the warp's tokens, in the step
    const int mine = team.run % kWarpRuns * T;                                  // of the run's, among them
    const TileX xt(p.x, w, column, p.c - column, first), ot(p.o, w, column, p.c - column, first);
    const TileG gt(p.g, w, column, p.c - column, first);
    const uint32_t space = shared_address(tiles) + threadIdx.x / 32 * kTileSteps * kTile;
    const uint32_t x_run = mine * TileX::kRow + team.lane * 2 * sizeof(TX);
    const uint32_t g_run = TileX::kBytes + mine * TileG::kRow + team.lane * 2 * sizeof(TG);
    const int cell = team.run * LPR + team.lane;
    auto bring = [&](int step, uint32_t tile) {
      const long long token = static_cast<long long>(step) * span;
      const int left = step < steps ? p.n - step * span - first : 0;
      xt.copy(tile, xt.step(p.x, token), left);
      gt.copy(tile + TileX::kBytes, gt.step(p.g, token), left);
      copies_end();
    };
    // The first walk: the run's sum from zero, and of its gates. True where one of them may be minus infinity.
    auto sum_up = [&](int step, uint32_t tile) {
      float2 sum = make_float2(0.f, 0.f), h = sum;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const float2 gv = unpack_pair<TG>(TileG::get(tile + g_run, t));
        sum = add2(sum, gv);
        h = fma2(decay<TX>(gv), h, unpack_pair<TX>(TileX::get(tile + x_run, t)));
      }
      const bool drops = __any_sync(0xffffffffu, may_drop(sum));
      if (drops && __any_sync(0xffffffffu, no_number(sum))) {
#pragma unroll 1
        for (int t = 0; t < T; ++t) mark_drops(unpack_pair<TG>(TileG::get(tile + g_run, t)), &sum);
      }
      if (spoilt(drops, h)) {
        h = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int t = 0; t < T; ++t)
          h = advance<TX, true>(unpack_pair<TG>(TileG::get(tile + g_run, t)), h, unpack_pair<TX>(TileX::get(tile + x_run, t)));
      }
      const JoinSpace j = join_space<LPR>(after_tiles, step & 1);
      j.run[cell] = run_map(sum, h);
      j.before[cell] = sum;
      hand_over(kMapsReady + (step & 1));
      return drops;
    };
    bring(0, space);
    bring(1, space + kTile);
    bring(2, space + 2 * kTile);
    if (team.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
    uint32_t tile = space, next = space + kTile, last = space + 2 * kTile;
    copies_wait<2>();
    bool drops = sum_up(0, tile);
    for (int step = 0; step < steps; ++step) {
      bool next_drops = false;
      copies_wait<1>();
      if (step + 1 < steps) next_drops = sum_up(step + 1, next);
      take_over(kStatesReady + (step & 1));
      float2 h = join_space<LPR>(after_tiles, step & 1).before[cell];
      const int t0 = step * span + first + mine;
      if (p.states != nullptr && t0 < p.n)
        store_pair<float, PIECE == 16>(p.states + state_of(p, w, t0 / T, runs_all), 1, w.ok0, w.ok1, h);
      // (all rows first: each load behind the store of the token before made the walk twice as long)
      typename PairOf<TX>::Raw x[T];
      float2 a[T];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        x[t] = TileX::get(tile + x_run, t);
        a[t] = decay<TX>(unpack_pair<TG>(TileG::get(tile + g_run, t)));
      }
      const float2 start = h;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        h = fma2(a[t], h, unpack_pair<TX>(x[t]));
        TileX::put(tile + x_run, t, h);
      }
      if (spoilt(drops, h)) {
        const InMemory<typename PairOf<TX>::Raw, T> xm(x);
        h = start;
#pragma unroll 1
        for (int t = 0; t < T; ++t) {
          h = advance<TX, true>(unpack_pair<TG>(TileG::get(tile + g_run, t)), h, unpack_pair<TX>(xm.v[t]));
          TileX::put(tile + x_run, t, h);
        }
      }
      __syncwarp();
      ot.store(tile, ot.step(p.o, static_cast<long long>(step) * span), p.n - step * span - first);
      __syncwarp();
      bring(step + kTileSteps, tile);
      const uint32_t free = tile;
      tile = next;
      next = last;
      last = free;
      drops = next_drops;
    }
  }
  if (team.ranks > 1) cg::this_cluster().sync();  // (nobody leaves while a peer that gave up early may still be written to)
}

template <typename TX, typename TG, int LPR, int PIECE>
__global__ void __launch_bounds__(kTileThreads, 2) fla_recurrence_bwd_kernel(const RecurrenceParams p) {
  constexpr int T = kRunTokens<TX, TG>, kRuns = kTileThreads / LPR, kWarpRuns = 32 / LPR;
  using TileX = WarpTile<TX, LPR, T, PIECE>;
  using TileG = WarpTile<TG, LPR, T, PIECE>;
  extern __shared__ uint4 tiles[];
  __shared__ RecurrenceShared<LPR, kTileThreads> sh;
  Team team;
  Place w;
  take_place<true, LPR>(p, sh.arrived, &team, &w);
  bool lost = false;
  const int column = w.c0 - 2 * team.lane;
  const int span = team.ranks * kRuns;                        // runs a step
  const int nth = span - 1 - (team.rank * kRuns + team.run);  // of the step's runs, in the order of the tokens
  const int first = nth / kWarpRuns * kWarpRuns * T, mine = nth % kWarpRuns * T;
  // (a tensor that is not there has no columns: nothing is copied, its rows are zero)
  const RecurrenceTensor& dy = p.o.ptr != nullptr ? p.o : p.x;
  const TileX xt(p.x, w, column, p.c - column, first), yt(dy, w, column, p.o.ptr != nullptr ? p.c - column : 0, first);
  const TileX dxt(p.dx, w, column, p.dx.ptr != nullptr ? p.c - column : 0, first);
  const TileG gt(p.g, w, column, p.c - column, first), dgt(p.dg, w, column, p.dg.ptr != nullptr ? p.c - column : 0, first);
  const uint32_t space = shared_address(tiles) + threadIdx.x / 32 * kBwdTile<TX, TG, LPR>;
  const uint32_t y_at = space + TileX::kBytes, dx_at = space + 2 * TileX::kBytes, g_at = space + 3 * TileX::kBytes, dg_at = g_at + TileG::kBytes;
  const uint32_t x_run = mine * TileX::kRow + team.lane * 2 * sizeof(TX), g_run = mine * TileG::kRow + team.lane * 2 * sizeof(TG);
  const long long cell = static_cast<long long>(w.b * p.heads + w.h) * p.c + w.c0;
  float2 carry = make_float2(0.f, 0.f);
  if (team.run == 0 && p.start != nullptr) carry = load_pair<float, PIECE == 16>(p.start + cell, 1, w.ok0, w.ok1);

  const int runs_all = (p.n - 1) / T + 1;
  const int steps = (runs_all - 1) / span + 1;
  float2 state;
  auto bring = [&](int step) {
    const long long token = static_cast<long long>(step) * span * T;
    const int left = step >= 0 ? static_cast<int>(p.n - token) - first : 0;
    xt.copy(space, xt.step(p.x, token), left);
    yt.copy(y_at, yt.step(dy, token), left);
    gt.copy(g_at, gt.step(p.g, token), left);
    copies_end();
    state = make_float2(0.f, 0.f);
    const int run = step * span + nth;
    if (step >= 0 && run < runs_all)
      state = load_pair<float, PIECE == 16>(p.states + state_of(p, w, run, runs_all), 1, w.ok0, w.ok1);
  };
  bring(steps - 1);
  if (team.ranks > 1) cg::this_cluster().sync();  // every CTA has started before a peer writes to it
  // The walk starts at the end; the runs behind the last token are the identity.
  for (int step = steps - 1; step >= 0; --step) {
    typename PairOf<TX>::Raw y[T];
    typename PairOf<TG>::Raw g[T];
    copies_wait<0>();
    float2 sum = make_float2(0.f, 0.f), r = sum, h = state;
    float2 a = sum;
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      y[t] = TileX::get(y_at + x_run, t);
      g[t] = TileG::get(g_at + g_run, t);
      const float2 gv = unpack_pair<TG>(g[t]);
      sum = add2(sum, gv);
      r = t == T - 1 ? unpack_pair<TX>(y[t]) : fma2(a, r, unpack_pair<TX>(y[t]));
      a = decay<TX>(gv);
    }
    r = mul2(a, r);
    const bool drops = __any_sync(0xffffffffu, may_drop(sum));
    if (drops && __any_sync(0xffffffffu, no_number(sum))) {
#pragma unroll 1
      for (int t = 0; t < T; ++t) mark_drops(unpack_pair<TG>(TileG::get(g_at + g_run, t)), &sum);
    }
    float2 before[T];  // the state before each token
    anew(g);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      before[t] = h;
      h = advance<TX, false>(unpack_pair<TG>(g[t]), h, unpack_pair<TX>(TileX::get(space + x_run, t)));
    }
    if (spoilt(drops, r)) {
      const InMemory<typename PairOf<TX>::Raw, T> ym(y);
      const InMemory<typename PairOf<TG>::Raw, T> gm(g);
      r = retreat_from_zero<TX, TG, T>(ym.v, gm.v);
    }
    const bool states_spoilt = spoilt(drops, h);
    if (states_spoilt) {
      const InMemory<typename PairOf<TG>::Raw, T> gm(g);
      float2 bm[T];
      h = state;
#pragma unroll 1
      for (int t = 0; t < T; ++t) {
        bm[t] = h;
        h = advance<TX, true>(unpack_pair<TG>(gm.v[t]), h, unpack_pair<TX>(TileX::get(space + x_run, t)));
      }
#pragma unroll
      for (int t = 0; t < T; ++t) before[t] = bm[t];
    }
    __syncwarp();  // every lane has its rows: the tiles are free
    bring(step - 1);
    r = exchange(sh, steps - 1 - step, sum, r, team, p, carry, lost);
    anew(y);
    anew(g);
    const float2 start = r;
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      const float2 all = t == T - 1 ? add2(unpack_pair<TX>(y[t]), r) : fma2(a, r, unpack_pair<TX>(y[t]));
      TileX::put(dx_at + x_run, t, all);
      a = decay<TX>(unpack_pair<TG>(g[t]));
      TileG::put(dg_at + g_run, t, mul2(mul2(a, all), before[t]));
      r = all;
    }
    if (states_spoilt || spoilt(drops, mul2(a, r))) {
      const InMemory<typename PairOf<TX>::Raw, T> ym(y);
      const InMemory<typename PairOf<TG>::Raw, T> gm(g);
      const InMemory<float2, T> bm(before);
      r = start;
#pragma unroll 1
      for (int t = T - 1; t >= 0; --t) {
        const float2 yv = unpack_pair<TX>(ym.v[t]), gv = unpack_pair<TG>(gm.v[t]);
        const float2 all = t == T - 1 ? add2(yv, r) : advance<TX, true>(unpack_pair<TG>(gm.v[t + 1]), r, yv);
        TileX::put(dx_at + x_run, t, all);
        float2 d = mul2(mul2(decay<TX>(gv), all), bm.v[t]);
        if (gv.x == -INFINITY) d.x = 0.f;
        if (gv.y == -INFINITY) d.y = 0.f;
        TileG::put(dg_at + g_run, t, d);
        r = all;
      }
    }
    __syncwarp();
    const long long token = static_cast<long long>(step) * span * T;
    const int left = static_cast<int>(p.n - token) - first;
    dxt.store(dx_at, dxt.step(p.dx, token), left);
    dgt.store(dg_at, dgt.step(p.dg, token), left);
    __syncwarp();
  }
  if (p.end != nullptr && team.run == 0 && team.rank == 0) store_pair<float, PIECE == 16>(p.end + cell, 1, w.ok0, w.ok1, carry);
  if (team.ranks > 1) cg::this_cluster().sync();  // (nobody leaves while a peer that gave up early may still be written to)
}

}  // namespace fla

namespace {

using fla::RecurrenceParams;
using fla::RecurrenceTensor;

constexpr int kShortTokens = 32;  // sequences up to here have nothing to exchange

int element_bytes(int dtype) { return dtype == FLA_DTYPE_F32 ? 4 : 2; }

// The call as the kernels see it. Channels of all heads (and, for one token, of the batch) that lie next to each
// other in every tensor are one row: narrow heads then fill a warp.
struct Plan {
  RecurrenceParams p;
  bool pair;        // two neighbouring columns can be read at once in every tensor
  int piece;        // bytes that rows can be copied in: 16, 4, or 0
  int lpr;
  int batch;
  long long farthest;  // bytes from one token to the next, of the tensor where they are most
};

void add_tensor(const FlaTensor& t, RecurrenceTensor* out) {
  out->ptr = t.ptr;
  out->sb = t.stride_b;
  out->sh = t.stride_h;
  out->sn = t.stride_n;
}

Plan make_plan(const FlaRecurrenceArgs* a, bool backward, int sm_count) {
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
  p.status = a->status;
  p.wait_limit_ns = (a->wait_limit_us ? a->wait_limit_us : 2000000ull) * 1000ull;
  p.withhold = (a->debug_flags & FLA_DEBUG_WITHHOLD_FIRST_TILE) != 0;
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
      if (all[i]->ptr != nullptr) ok = holds(*all[i], sizes[i]) && ok;
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
  const long long columns = p.c;  // (up to 2^30: what is formed from it passes 32 bits)
  auto rows_on = [&](int bytes) {
    return columns * sizes[0] % bytes == 0 && columns * sizes[1] % bytes == 0 && every([&](const RecurrenceTensor& t, int size) {
             return reinterpret_cast<uintptr_t>(t.ptr) % bytes == 0 && (p.n == 1 || t.sn * size % bytes == 0) &&
                    (p.heads == 1 || t.sh * size % bytes == 0) && (plan.batch == 1 || t.sb * size % bytes == 0);
           });
  };
  plan.piece = plan.pair && rows_on(16) ? 16 : rows_on(4) ? 4 : 0;
  plan.farthest = 1;
  every([&](const RecurrenceTensor& t, int size) {
    plan.farthest = std::max(plan.farthest, t.sn < 0 ? INT64_MAX : t.sn * size);  // (backwards: alone, too, where offsets have a sign)
    return true;
  });
  // Tiles of 64 columns; of 32 where that leaves fewer lanes without one, and for few channels, whose clusters of eight would
  // leave places on the SMs empty. Microseconds forward + backward with tiles of 64 and 32: 8 x 128 channels, 65536 tokens, bf16
  // 215 + 306 / 128 + 214, fp32 403 + 531 / 204 + 303; 4 x 256 channels, 8192 tokens 38 + 44 / 23 + 34; but 32 x 128 channels,
  // 2048 tokens 19 + 27 / 19 + 32, and 128 x 64 channels, 4096 tokens 48 + 82 / 52 + 89.
  const long long tiles64 = (columns + 63) / 64 * p.heads * plan.batch;
  plan.lpr = (columns + 31) / 32 * 32 * 10 < (columns + 63) / 64 * 64 * 9 || tiles64 * fla::kRecMaxCluster <= 2 * sm_count ? 16 : 32;
  p.tiles = static_cast<int>((columns + 2 * plan.lpr - 1) / (2 * plan.lpr));
  p.tiles_all = static_cast<long long>(p.tiles) * p.heads * plan.batch;
  return plan;
}

// CTAs of a cluster and threads of a CTA (that work on runs). A tile of channels is walked by one cluster from end to end;
// more CTAs, and larger ones, walk it in fewer steps, of which each takes longer.
struct Shape {
  int threads, ranks;
};
Shape shape_of(const Plan& plan, int run_tokens, bool backward, bool two_resident, int sm_count) {
  const long long runs = (plan.p.n - 1) / run_tokens + 1;
  Shape s = {256, 1};
  auto step = [&] { return static_cast<long long>(s.ranks) * s.threads / plan.lpr; };
  if (plan.piece) {
    // Backward two CTAs an SM. Forward two where their tiles are small enough (16-bit rows with fp32 gates), else one in a
    // cluster: its CTAs all have to be there at once.
    const int most = backward || two_resident ? 2 * sm_count : sm_count;
    while (s.ranks < fla::kRecMaxCluster && plan.p.tiles_all * s.ranks * 2 <= most && step() < runs) s.ranks *= 2;
    return s;
  }
  while (s.ranks < fla::kRecMaxCluster && plan.p.tiles_all * s.ranks < 2 * sm_count && step() < runs) s.ranks *= 2;
  if (plan.p.tiles_all * s.ranks <= sm_count && step() < runs) s.threads = backward ? 512 : 1024;
  return s;
}

template <typename TX, typename TG, int LPR>
int launch(const Plan& plan, bool backward, int sm_count, cudaStream_t stream) {
  constexpr int T = fla::kRunTokens<TX, TG>;
  constexpr int kFwdBytes = fla::kTileThreads / 32 * fla::kTileSteps * fla::kFwdTile<TX, TG, LPR> + fla::kJoinBytes<LPR>;
  constexpr bool kTwoResident = kFwdBytes + fla::kTradeBytes<LPR> + 1024 <= 228 * 1024 / 2;
  Shape shape = shape_of(plan, T, backward, kTwoResident, sm_count);
  const bool alone = plan.p.n <= kShortTokens || plan.farthest > 0x7fffffffLL / (shape.ranks * (shape.threads / LPR) * T);
  long long blocks = plan.p.tiles_all * shape.ranks;
  if (alone) {
    shape = {fla::kShortThreads, 1};
    blocks = (plan.p.tiles_all * LPR + shape.threads - 1) / shape.threads;
  }
  if (blocks > 0x7fffffffLL) return FLA_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(shape.threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = shape.ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = shape.ranks > 1 ? 1 : 0;
  auto go = [&](auto kernel, const char* name) {
    if (cfg.dynamicSmemBytes > 0 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                         static_cast<int>(cfg.dynamicSmemBytes)) != cudaSuccess)
      return static_cast<int>(FLA_ERR_CUDA);
    return fla::launched(cudaLaunchKernelEx(&cfg, kernel, plan.p), name);
  };
  if (alone)
    return plan.pair ? (backward ? go(fla::fla_recurrence_short_bwd_kernel<TX, TG, true, LPR>, "fla_recurrence_short_bwd_kernel")
                                 : go(fla::fla_recurrence_short_fwd_kernel<TX, TG, true, LPR>, "fla_recurrence_short_fwd_kernel"))
                     : (backward ? go(fla::fla_recurrence_short_bwd_kernel<TX, TG, false, LPR>, "fla_recurrence_short_bwd_kernel")
                                 : go(fla::fla_recurrence_short_fwd_kernel<TX, TG, false, LPR>, "fla_recurrence_short_fwd_kernel"));
  if (plan.piece) {
    if (backward) {
      cfg.dynamicSmemBytes = fla::kTileThreads / 32 * fla::kBwdTile<TX, TG, LPR>;
      return plan.piece == 16 ? go(fla::fla_recurrence_bwd_kernel<TX, TG, LPR, 16>, "fla_recurrence_bwd_kernel")
                              : go(fla::fla_recurrence_bwd_kernel<TX, TG, LPR, 4>, "fla_recurrence_bwd_kernel");
    }
    cfg.blockDim = dim3(fla::kTileThreads + 32);
    cfg.dynamicSmemBytes = kFwdBytes + (shape.ranks > 1 ? fla::kTradeBytes<LPR> : 0);
    return plan.piece == 16 ? go(fla::fla_recurrence_fwd_kernel<TX, TG, LPR, 16>, "fla_recurrence_fwd_kernel")
                            : go(fla::fla_recurrence_fwd_kernel<TX, TG, LPR, 4>, "fla_recurrence_fwd_kernel");
  }
  if constexpr (sizeof(TX) == 4) {
    return FLA_ERR_UNSUPPORTED;  // (fp32 rows always lie on 4 bytes)
  } else {
    if (shape.threads == 256)
      return backward ? go(fla::fla_recurrence_direct_bwd_kernel<TX, TG, LPR, 256>, "fla_recurrence_direct_bwd_kernel")
                      : go(fla::fla_recurrence_direct_fwd_kernel<TX, TG, LPR, 256>, "fla_recurrence_direct_fwd_kernel");
    return backward ? go(fla::fla_recurrence_direct_bwd_kernel<TX, TG, LPR, 512>, "fla_recurrence_direct_bwd_kernel")
                    : go(fla::fla_recurrence_direct_fwd_kernel<TX, TG, LPR, 1024>, "fla_recurrence_direct_fwd_kernel");
  }
}

template <typename TX, typename TG>
int launch_types(const Plan& plan, bool backward, int sm_count, cudaStream_t stream) {
  return plan.lpr == 16 ? launch<TX, TG, 16>(plan, backward, sm_count, stream) : launch<TX, TG, 32>(plan, backward, sm_count, stream);
}

bool known_type(int t) { return t == FLA_DTYPE_BF16 || t == FLA_DTYPE_F16 || t == FLA_DTYPE_F32; }

int check(const FlaRecurrenceArgs* a) {
  if (a == nullptr || a->batch <= 0 || a->heads <= 0 || a->seqlen <= 0 || a->dim <= 0) return FLA_ERR_INVALID;
  if (!known_type(a->dtype) || (a->g_dtype != a->dtype && a->g_dtype != FLA_DTYPE_F32)) return FLA_ERR_INVALID;
  if (a->x.ptr == nullptr || a->g.ptr == nullptr) return FLA_ERR_INVALID;
  // run, token and column numbers are 32-bit, a step or a tile past the end included
  if (a->seqlen > (1 << 30) || a->dim > (1 << 30) || static_cast<long long>(a->batch) * a->heads > (1 << 30)) return FLA_ERR_UNSUPPORTED;
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
  const Plan plan = make_plan(a, backward, sm_count);
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
