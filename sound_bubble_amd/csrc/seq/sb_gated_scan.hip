// Gated linear recurrence over the middle axis of [outer, steps, inner]:  h_t = a_t h_{t-1} + b_t, forward, backward, one step.
//
// Steps are joined as pairs (A, B): h -> A h + B; (A2, B2) after (A1, B1) is (A2 A1, A2 B1 + B2).  A lane holds one channel of one
// sequence, S consecutive steps of it in registers, and all lanes of a wave are at the same steps, so that a step's address and what
// is live are the wave's business and nothing goes over lanes.  The waves of a workgroup are consecutive in time; their pairs meet
// in LDS, where every wave joins them in the same order, and the state is carried from chunk to chunk by the same workgroup: x and gate
// are read once and the order of all products is fixed by the sizes.  Where there are too few channels to fill the chip, time is cut
// into segments: a first kernel makes each segment's pair, the second joins those in front of its own.
// Steps that a sequence does not have (behind its length, behind the last chunk) are (1, 0) by selection, whatever memory holds.
//
// The backward pass makes h_{t-1} again in fp32 from the states the forward pass left in front of every chunk, and walks
//   G_t = dh_t + c_{t+1},  c_t = a_t G_t
// down the same chunks: the pairs are (A, D): c -> A c + D, with A the forward pass's product.
#include <cmath>

#include "sb_seq_common.h"

namespace {

// Steps a lane holds, and waves of a workgroup (which then has 256 registers a lane).  bf16 8 x 4096 x 2048, forward / backward, us: 16 x 8
// 98 / 160, 8 x 16 108 / 176, 8 x 8 111 / 162; two channels a lane: 179 / 250 (half the workgroups, twice the registers).
constexpr int S = 16, kMaxWaves = 8;
// Workgroups with fewer waves than kFewWaves in all leave the chip half empty: time is cut so that there are about kWaves.  That reads x and
// gate twice.  fp16 6 x 3001 x 1000 (752 waves) forward / backward, us: cut 68 / 94, whole 94 / 134.
// A segment joins the pairs of all in front of it, 0.1 us each, and walks its own chunks, 2.4 us each in both kernels: of c chunks about
// 5 sqrt(c) segments.  fp32 1 x 262144 x 16 forward / backward, us: 64 segments 217 / 258, 226 87 / 106; 1 x 65536 x 64: 64 49 / 56, 113 40 / 45.
// (409 segments: their pairs and powers take what 512 pairs do)
constexpr int kFewWaves = 1024, kWaves = 4096, kMaxSplits = 409;

struct Lay {
  int nw, splits;                  // waves along time, segments of time
  int64_t tiles;                   // workgroups' channel tiles: 64 lanes of the flattened (sequence, channel) axis
  int64_t steps, chunks;           // steps of a chunk, chunks of a sequence
};

Lay lay_of(int64_t outer, int64_t steps, int64_t inner) {
  Lay l;
  l.tiles = (outer * inner + 63) / 64;
  l.nw = 1;
  // (more waves along time until there are 8 a SIMD: fp32 16 x 625 x 4640 forward 115 us, with half as many 123)
  while (l.nw < kMaxWaves && l.nw * S < steps && l.tiles * l.nw < 8192) l.nw *= 2;
  l.steps = (int64_t)l.nw * S;
  l.chunks = (steps + l.steps - 1) / l.steps;
  l.splits = 1;
  const int64_t waves = l.tiles * l.nw;
  if (waves < kFewWaves && l.chunks >= 4) {
    const int64_t most = std::min<int64_t>(kMaxSplits, std::min<int64_t>(l.chunks / 2, (int64_t)(5 * std::sqrt((double)l.chunks))));
    l.splits = (int)std::min<int64_t>(most, kWaves / waves);
  }
  return l;
}

struct Kargs {
  int64_t outer, steps, inner, chunks, chunk_steps;
  int reverse, splits;
  const void* x; int64_t so_x, st_x;
  const void* gate; int64_t so_g, st_g;
  const void* dh; int64_t so_d, st_d;
  const float* h0; const float* dlast; const int64_t* len;
  void* h; float* h_last; float* states; float* agg;
  void* dx; void* dgate; float* dh0;
};

// a = s(z) and 1 - a without cancellation: e = exp(-|z|) as 2^(hi + lo), s(|z|) = 1 / (1 + e).  Behind |z| = 87 e is below the normal
// numbers (and the exponential unit gives 0 for those): it counts as 0, so that infinite gates are exactly 0 and 1.
SB_DEVINL void logistic(float z, float& a, float& one_less) {
  const float az = __builtin_fabsf(z);
  const float t = az * SB_NLOG2E;
  const float lo = __builtin_fmaf(az, SB_NLOG2E, -t) + az * -1.925963033500e-8f;      // -log2(e) - (float) -log2(e)
  float e = __builtin_amdgcn_exp2f(t);
  e = az > 87.f ? 0.f : __builtin_fmaf(e, lo * 0.69314718f, e);                       // (infinite z: lo is NaN)
  const float r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
  const bool pos = z >= 0.f;
  a = pos ? r : q;
  one_less = pos ? q : r;
}

// where a lane stands
struct Place {
  int wave, waves;
  bool on;                                // the lane has a channel
  int64_t q, o, c, lo, hi;                // flattened channel, sequence, channel, live steps [lo, hi) in the order of the walk
  int64_t all_lo, all_hi;                 // steps that are live in every lane of the wave (uniform)
  SB_DEVINL Place(const Kargs& k) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    waves = blockDim.x >> 6;
    q = ((int64_t)blockIdx.x * 64 + (threadIdx.x & 63));
    on = q < k.outer * k.inner;
    o = on ? q / k.inner : 0;
    c = on ? q - o * k.inner : 0;
    q = on ? q : 0;
    int64_t n = on ? k.steps : 0;
    if (on && k.len) n = min(max(k.len[o], (int64_t)0), k.steps);
    lo = k.reverse ? k.steps - n : 0;
    hi = k.reverse ? k.steps : n;
    all_lo = lo;
    all_hi = hi;
    if (!__all(on && n == k.steps)) {
      for (int d = 1; d < 64; d *= 2) {
        all_lo = max(all_lo, (int64_t)__shfl_xor((long long)all_lo, d, 64));
        all_hi = min(all_hi, (int64_t)__shfl_xor((long long)all_hi, d, 64));
      }
    }
    all_lo = first(all_lo);
    all_hi = __all(on) ? first(all_hi) : 0;
  }
  static SB_DEVINL int64_t first(int64_t v) {
    return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
  }
  // live steps of the lane's S from t on, as a bit each
  SB_DEVINL unsigned live(int64_t t) const {
    const int n0 = (int)min(max(lo - t, (int64_t)0), (int64_t)S), n1 = (int)min(max(hi - t, (int64_t)0), (int64_t)S);
    return ((1u << n1) - 1u) & ~((1u << n0) - 1u);
  }
  SB_DEVINL bool full(int64_t t) const { return t >= all_lo && t + S <= all_hi; }
};

template <class E> SB_DEVINL void load_steps(E (&v)[S], const void* base, int64_t so, int64_t st, const Place& p, const Kargs& k, int64_t t, bool full,
                                             unsigned live) {
  const int64_t step = k.reverse ? -st : st;
  const E* at = (const E*)base + (k.reverse ? k.steps - 1 - t : t) * st + p.o * so + p.c;
  if (full) {
#pragma unroll
    for (int s = 0; s < S; ++s, at += step) v[s] = *at;
  } else {
#pragma unroll
    for (int s = 0; s < S; ++s, at += step) {
      v[s] = (E)0.f;
      if (live >> s & 1) v[s] = *at;
    }
  }
}
template <class E> SB_DEVINL void store_steps(void* base, const E (&v)[S], const Place& p, const Kargs& k, int64_t t, bool full) {
  const int64_t step = k.reverse ? -k.inner : k.inner;
  E* at = (E*)base + ((k.reverse ? k.steps - 1 - t : t) + p.o * k.steps) * k.inner + p.c;
  if (full) {
#pragma unroll
    for (int s = 0; s < S; ++s, at += step) *at = v[s];
  } else if (p.on) {
#pragma unroll
    for (int s = 0; s < S; ++s, at += step)
      if (t + s < k.steps) *at = v[s];
  }
}

// Everything this wave has under way has arrived.  In front of a loop whose loads wait by count for one round: without it the counts
// have to allow for what was issued on the way in, and the loop would wait for its own stores.
SB_DEVINL void wait_memory() {
  __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0)
}
// a barrier that leaves loads and stores under way: the waves exchange nothing but LDS
SB_DEVINL void block_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);      // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// a_t and what multiplies x_t
template <int FORM> SB_DEVINL void coefficients(float g, float& a, float& ol) {
  if constexpr (FORM == SB_SCAN_SIGMOID) {
    logistic(g, a, ol);
  } else {
    a = g;
    ol = 1.f;
  }
}
SB_DEVINL void kill_dead(float (&a)[S], float (&ol)[S], unsigned live) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    a[s] = live >> s & 1 ? a[s] : 1.f;
    ol[s] = live >> s & 1 ? ol[s] : 0.f;
  }
}
template <class E> SB_DEVINL void kill_dead(E (&v)[S], unsigned live) {
#pragma unroll
  for (int s = 0; s < S; ++s) v[s] = live >> s & 1 ? v[s] : (E)0.f;
}

// The product of a segment's gates leaves float32 where they are beyond 1 ("decay": 256 gates of 1.5 are 2^150), and an infinite product times
// a state of 0 is NaN where the recurrence stays 0.  It is kept as A 2^power, 0.5 <= |A| < 1 (or 0, infinite, NaN, power whatever), which
// rounds as the product itself does; the power is taken out every S gates, so that only products of S have to stay within float32.
SB_DEVINL void take_power(float& A, int& power) {
  power += __builtin_amdgcn_frexp_expf(A);      // (at most 2400 for S gates: 2^31 is 14 M steps of a wave, 10^10 elements and more)
  A = __builtin_amdgcn_frexp_mantf(A);
}
SB_DEVINL bool is_normal(int power) { return power >= -125 && power <= 128; }
// A 2^power c + B; one rounding where A 2^power is a normal number
SB_DEVINL float join_power(float A, int power, float c, float B) {
  if (is_normal(power)) return __builtin_fmaf(__builtin_ldexpf(A, power), c, B);
  return __builtin_ldexpf(A * c, power) + B;
}
// As it is kept for the second kernel: the product itself where that is a normal number, 0, infinite or NaN.  Where not, its mantissa as the bits
// of a subnormal number, which nothing else is then (a power of two gets an ulp), with the power beside it.  Behind 1000 any state but 0 is
// infinite; below 2^-278 any finite one is 0, and so is the product: most of the segments of a sequence that decays.
// (bf16 1 x 131072 x 512 with fp32 gates, second kernel forward / backward: 97 / 171 us, where powers are read for every segment 101 / 181.)
constexpr unsigned kSign = 0x80000000u, kFraction = 0x007FFFFFu, kHalf = 126u << 23;
SB_DEVINL bool is_far(float kept) { return __builtin_amdgcn_classf(kept, 0x90); }      // (subnormal, either sign)
SB_DEVINL float keep_power(float A, int power, int16_t* at) {
  const unsigned bits = (unsigned)__float_as_int(A);
  if (is_normal(power) || (bits & ~(kSign | kFraction)) != kHalf) return __builtin_ldexpf(A, power);
  if (power <= -278) return 0.f;
  *at = (int16_t)min(power, 1000);
  return __int_as_float((int)((bits & kSign) | max(bits & kFraction, 1u)));
}
SB_DEVINL float join_kept(float kept, int power, float c, float B) {
  const float near = __builtin_fmaf(kept, c, B);
  const float A = __int_as_float((int)((unsigned)__float_as_int(kept) | kHalf));
  return is_far(kept) ? __builtin_ldexpf(A * c, power) + B : near;
}

// the pairs of a workgroup's waves, two buffers in turn: [turn][wave][lane]
struct Pairs {
  float2* lds;
  int waves;
  SB_DEVINL float2& at(int turn, int wave) const { return lds[(turn * waves + wave) * 64 + (threadIdx.x & 63)]; }
  // carry over all waves; in: what enters wave `mine`
  template <bool UP> SB_DEVINL void join(int turn, int mine, float& carry, float& in) const {
    for (int w = 0; w < waves; ++w) {
      const int j = UP ? w : waves - 1 - w;
      const float2 r = at(turn, j);
      if (j == mine) in = carry;
      carry = __builtin_fmaf(r.x, carry, r.y);
    }
  }
  SB_DEVINL float product(int turn) const {
    float v = 1.f;
    for (int w = 0; w < waves; ++w) v *= at(turn, w).x;
    return v;
  }
};

// k.agg: the segments' pairs [split][A | B][plane], then ("decay") the powers [split][plane] of products that are far, in 16 bits
SB_DEVINL int16_t* powers_of(const Kargs& k) { return (int16_t*)(k.agg + 2 * k.splits * k.outer * k.inner); }
int64_t pairs_floats(int64_t splits, int64_t plane) { return 2 * (splits + (splits + 3) / 4) * plane; }

// state in front of segment `split`: h0 and the pairs of the earlier ones (UP), dlast and those of the later ones (!UP)
template <int FORM, bool UP> SB_DEVINL float fold_splits(const float* start, const Place& p, const Kargs& k, int split) {
  const int64_t plane = k.outer * k.inner;
  if (!p.on) return 0.f;
  float carry = start ? start[p.q] : 0.f;
  const int n = UP ? split : k.splits - 1 - split;
  const unsigned at = (unsigned)p.q;      // (time is cut where there are fewer than 2^16 channels)
  constexpr int N = 16;
  for (int j0 = 0; j0 < n; j0 += N) {      // (the loads of N pairs at once: one after the other they cost a trip to memory each)
    float A[N], B[N];
    bool far = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = UP ? j0 + i : k.splits - 1 - j0 - i;
      A[i] = j0 + i < n ? (k.agg + (2 * j) * plane)[at] : 1.f;
      B[i] = j0 + i < n ? (k.agg + (2 * j + 1) * plane)[at] : 0.f;
    }
    if constexpr (FORM == SB_SCAN_DECAY) {
#pragma unroll
      for (int i = 0; i < N; ++i) far |= is_far(A[i]);
    }
    if (__any(far)) {      // (read again, four at a time: 16 with their powers cost the kernel registers, and with them waves)
#pragma unroll 1
      for (int j1 = j0; j1 < min(j0 + N, n); j1 += 4) {
        float a[4], b[4];
        int power[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = UP ? min(j1 + i, n - 1) : k.splits - 1 - min(j1 + i, n - 1);
          a[i] = (k.agg + (2 * j) * plane)[at];
          b[i] = (k.agg + (2 * j + 1) * plane)[at];
          power[i] = (powers_of(k) + j * plane)[at];      // (of one that is not far: whatever is there)
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) carry = j1 + i < n ? join_kept(a[i], power[i], carry, b[i]) : carry;
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (j0 + i < n) carry = __builtin_fmaf(A[i], carry, B[i]);
  }
  return carry;
}

// The pair of a segment of time: (A, B) of blockIdx.y from x and gate (UP), (A, D) of blockIdx.y + 1 from dh and gate.  The waves take
// consecutive parts of it, each by itself, and are joined once.
template <class T, class G, int FORM, bool UP>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_pair_kernel(Kargs k) {
  extern __shared__ float2 lds[];
  const Place p(k);
  const Pairs pairs{lds, p.waves};
  const int split = blockIdx.y + (UP ? 0 : 1);
  const int64_t g0 = k.chunks * split / k.splits * p.waves, groups = k.chunks * (split + 1) / k.splits * p.waves - g0;
  const int64_t first = (g0 + groups * p.wave / p.waves) * S, last = (g0 + groups * (p.wave + 1) / p.waves) * S - S;      // (>= one group a wave)
  const void* from = UP ? k.x : k.dh;
  const int64_t so = UP ? k.so_x : k.so_d, st = UP ? k.st_x : k.st_d, step = UP ? S : -S;
  float carry = 0.f, whole = 1.f;
  int power = 0;
  T x[S];
  G g[S];
#pragma unroll
  for (int s = 0; s < S; ++s) x[s] = (T)0.f;
  const auto load = [&](int64_t t, bool full) __attribute__((always_inline)) {
    const unsigned live = full ? 0u : p.live(t);
    load_steps<G>(g, k.gate, k.so_g, k.st_g, p, k, t, full, live);
    if (full || from) load_steps<T>(x, from, so, st, p, k, t, full, live);
  };
  const auto group = [&](int64_t t, auto fast, bool more) __attribute__((always_inline)) {
    constexpr bool FAST = decltype(fast)::value;
    float a[S], ol[S], xf[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      a[s] = (float)g[s];
      xf[s] = (float)x[s];      // (dead steps were loaded as 0)
    }
    const bool full = FAST || p.full(t);
    const unsigned live = full ? 0u : p.live(t);
    if constexpr (FAST) load(t + step, true);
    else if (more) load(t + step, from && p.full(t + step));
#pragma unroll
    for (int s = 0; s < S; ++s) coefficients<FORM>(a[s], a[s], ol[s]);
    if (!full) kill_dead(a, ol, live);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int s = UP ? i : S - 1 - i;
      whole *= a[s];
      carry = UP ? __builtin_fmaf(a[s], carry, ol[s] * xf[s]) : a[s] * (xf[s] + carry);
    }
    if constexpr (FORM == SB_SCAN_DECAY) take_power(whole, power);
  };
  int64_t t = UP ? first : last;
  int64_t left = (last - first) / S + 1;
  load(t, from && p.full(t));
  for (; left > 0; --left, t += step) {
    wait_memory();
    if (from)
      for (; left > 1 && p.full(t) && p.full(t + step); --left, t += step) group(t, std::true_type(), true);
    group(t, std::false_type(), left > 1);
  }
  if (p.waves > 1) {
    pairs.at(0, p.wave) = make_float2(whole, carry);
    if constexpr (FORM == SB_SCAN_DECAY) pairs.at(1, p.wave).x = __int_as_float(power);
    block_sync();
    carry = 0.f;
    if constexpr (FORM == SB_SCAN_DECAY) {
      power = 0;
      for (int w = 0; w < p.waves; ++w) {
        const int j = UP ? w : p.waves - 1 - w;
        const float2 r = pairs.at(0, j);
        const int q = __float_as_int(pairs.at(1, j).x);
        carry = join_power(r.x, q, carry, r.y);
        power += q;
      }
    } else {
      float in;
      pairs.template join<UP>(0, -1, carry, in);
    }
    whole = pairs.product(0);
    if constexpr (FORM == SB_SCAN_DECAY) take_power(whole, power);
  }
  if (p.wave == 0 && p.on) {
    const int64_t plane = k.outer * k.inner;
    if constexpr (FORM == SB_SCAN_DECAY) whole = keep_power(whole, power, powers_of(k) + split * plane + p.q);
    k.agg[(2 * split) * plane + p.q] = whole;
    k.agg[(2 * split + 1) * plane + p.q] = carry;
  }
}

// h, states, h_last
template <class T, class G, int FORM>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_fwd_kernel(Kargs k) {
  extern __shared__ float2 lds[];
  const Place p(k);
  const Pairs pairs{lds, p.waves};
  const int split = blockIdx.y;
  const int64_t c0 = k.chunks * split / k.splits, c1 = k.chunks * (split + 1) / k.splits, plane = k.outer * k.inner;
  float carry = fold_splits<FORM, true>(k.h0, p, k, split);
  T x[S];
  G g[S];
  const auto load = [&](int64_t t, bool full) __attribute__((always_inline)) {
    const unsigned live = full ? 0u : p.live(t);
    load_steps<T>(x, k.x, k.so_x, k.st_x, p, k, t, full, live);
    load_steps<G>(g, k.gate, k.so_g, k.st_g, p, k, t, full, live);
  };
  const auto start = [&](int64_t ch) { return ch * k.chunk_steps + p.wave * S; };
  // FAST: this chunk and the next have all their steps in this wave
  const auto chunk = [&](int64_t ch, auto fast) __attribute__((always_inline)) {
    constexpr bool FAST = decltype(fast)::value;
    const int64_t t = start(ch);
    const bool full = FAST || p.full(t);
    const unsigned live = full ? 0u : p.live(t);
    float a[S], b[S], xf[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      xf[s] = (float)x[s];
      a[s] = (float)g[s];
    }
    if constexpr (FAST) load(t + k.chunk_steps, true);
    else if (ch + 1 < c1) load(t + k.chunk_steps, p.full(t + k.chunk_steps));
#pragma unroll
    for (int s = 0; s < S; ++s) coefficients<FORM>(a[s], a[s], b[s]);
    if (!full) kill_dead(a, b, live);
    float A, B;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      b[s] *= xf[s];      // (dead steps were loaded as 0)
      A = s ? A * a[s] : a[s];
      B = s ? __builtin_fmaf(a[s], B, b[s]) : b[s];
    }
    if (k.states && p.wave == 0 && p.on) k.states[ch * plane + p.q] = carry;
    float in;
    if (p.waves > 1) {
      pairs.at(ch & 1, p.wave) = make_float2(A, B);
      block_sync();
      pairs.template join<true>(ch & 1, p.wave, carry, in);
    } else {
      in = carry;
      carry = __builtin_fmaf(A, carry, B);
    }
    T out[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      in = __builtin_fmaf(a[s], in, b[s]);
      out[s] = (T)in;
    }
    if (!full) kill_dead<T>(out, live);
    store_steps<T>(k.h, out, p, k, t, full);
  };
  load(start(c0), p.full(start(c0)));
  for (int64_t ch = c0; ch < c1; ++ch) {
    wait_memory();
    for (; ch + 1 < c1 && p.full(start(ch)) && p.full(start(ch + 1)); ++ch) chunk(ch, std::true_type());
    chunk(ch, std::false_type());
  }
  if (p.wave == 0 && p.on && split == k.splits - 1) k.h_last[p.q] = carry;
}

// dx, dgate, dh0
template <class T, class G, int FORM>
__global__ __launch_bounds__(64 * kMaxWaves) void gated_scan_bwd_kernel(Kargs k) {
  extern __shared__ float2 lds[];
  const Place p(k);
  const Pairs down{lds, p.waves}, up{lds + 2 * 64 * p.waves, p.waves};
  const int split = blockIdx.y;
  const int64_t c0 = k.chunks * split / k.splits, c1 = k.chunks * (split + 1) / k.splits, plane = k.outer * k.inner;
  float carry = fold_splits<FORM, false>(k.dlast, p, k, split);
  T x[S], d[S];
  G g[S];
  float state = 0.f;
#pragma unroll
  for (int s = 0; s < S; ++s) d[s] = (T)0.f;
  const auto load = [&](int64_t ch, int64_t t, bool full, bool has) __attribute__((always_inline)) {
    const unsigned live = full ? 0u : p.live(t);
    load_steps<G>(g, k.gate, k.so_g, k.st_g, p, k, t, full, live);
    if (has) load_steps<T>(d, k.dh, k.so_d, k.st_d, p, k, t, full, live);
    load_steps<T>(x, k.x, k.so_x, k.st_x, p, k, t, full, live);
    if (p.on) state = k.states[ch * plane + p.q];
  };
  const auto start = [&](int64_t ch) { return ch * k.chunk_steps + p.wave * S; };
  const auto chunk = [&](int64_t ch, auto fast) __attribute__((always_inline)) {
    constexpr bool FAST = decltype(fast)::value;
    const int64_t t = start(ch);
    const bool full = FAST || p.full(t);
    const unsigned live = full ? 0u : p.live(t);
    float a[S], ol[S], xf[S], df[S], h = state;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      a[s] = (float)g[s];
      xf[s] = (float)x[s];      // (dead steps were loaded as 0)
      df[s] = (float)d[s];
    }
    if constexpr (FAST) load(ch - 1, t - k.chunk_steps, true, true);
    else if (ch > c0) load(ch - 1, t - k.chunk_steps, p.full(t - k.chunk_steps), k.dh != nullptr);
#pragma unroll
    for (int s = 0; s < S; ++s) coefficients<FORM>(a[s], a[s], ol[s]);
    if (!full) kill_dead(a, ol, live);
    float A, D, B;
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      A = s < S - 1 ? A * a[s] : a[s];
      D = a[s] * (s < S - 1 ? df[s] + D : df[s]);
    }
#pragma unroll
    for (int s = 0; s < S; ++s) B = s ? __builtin_fmaf(a[s], B, ol[s] * xf[s]) : ol[0] * xf[0];
    float in;
    if (p.waves > 1) {
      down.at(ch & 1, p.wave) = make_float2(A, D);
      up.at(ch & 1, p.wave) = make_float2(A, B);
      block_sync();
      for (int w = 0; w < p.wave; ++w) {
        const float2 r = up.at(ch & 1, w);
        h = __builtin_fmaf(r.x, h, r.y);
      }
      down.template join<false>(ch & 1, p.wave, carry, in);
    } else {
      in = carry;
      carry = __builtin_fmaf(A, carry, D);
    }
    float hb[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      hb[s] = h;
      h = __builtin_fmaf(a[s], h, ol[s] * xf[s]);
    }
    T dx[S];
    G dg[S];
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      const float gt = df[s] + in;
      in = a[s] * gt;
      if constexpr (FORM == SB_SCAN_SIGMOID) {
        const float vx = ol[s] * gt;
        dx[s] = (T)vx;
        dg[s] = (G)(vx * a[s] * (hb[s] - xf[s]));
      } else {
        dx[s] = (T)gt;
        dg[s] = (G)(gt * hb[s]);
      }
    }
    if (!full) {
      kill_dead<T>(dx, live);
      kill_dead<G>(dg, live);
    }
    store_steps<T>(k.dx, dx, p, k, t, full);
    store_steps<G>(k.dgate, dg, p, k, t, full);
  };
  load(c1 - 1, start(c1 - 1), p.full(start(c1 - 1)), k.dh != nullptr);
  for (int64_t ch = c1 - 1; ch >= c0; --ch) {
    wait_memory();
    if (k.dh)
      for (; ch > c0 && p.full(start(ch)) && p.full(start(ch - 1)); --ch) chunk(ch, std::true_type());
    chunk(ch, std::false_type());
  }
  if (p.wave == 0 && p.on && split == 0 && k.dh0) k.dh0[p.q] = carry;
}

template <class T, class G, int FORM>
__global__ __launch_bounds__(256) void gated_scan_step_kernel(const T* x, const G* gate, float* state, T* y, int64_t inner, int64_t ld_x,
                                                              int64_t ld_g, int64_t per_row, int64_t total) {
  constexpr int V = 4;
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (j >= total) return;
  const int64_t row = j / per_row, c = (j - row * per_row) * V;
  const int n = (int)min((int64_t)V, inner - c);
  const Vec<T, V> xv = vload_n<T, V>(x + row * ld_x + c, n);
  const Vec<G, V> gv = vload_n<G, V>(gate + row * ld_g + c, n);
  Vec<float, V> h = vload_n<float, V>(state + row * inner + c, n);
  Vec<T, V> o;
  float a[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) coefficients<FORM>((float)gv.v[i], a[i], b[i]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h.v[i] = __builtin_fmaf(a[i], h.v[i], b[i] * (float)xv.v[i]);
    o.v[i] = (T)h.v[i];
  }
  vstore_n<float, V>(state + row * inner + c, h, n);
  vstore_n<T, V>(y + row * inner + c, o, n);
}

// f(T*, G*, integral_constant<form>)
template <class F> int with_types(int xtype, int gtype, int form, F&& f) {
  if (gtype != xtype && gtype != SB_F32) return -1002;
  if (form != SB_SCAN_DECAY && form != SB_SCAN_SIGMOID) return -1003;
  return sb_with_type(xtype, [&](auto* x) -> int {
    const auto go = [&](auto* g) -> int {
      if (form == SB_SCAN_SIGMOID) return f(x, g, std::integral_constant<int, SB_SCAN_SIGMOID>());
      return f(x, g, std::integral_constant<int, SB_SCAN_DECAY>());
    };
    if (gtype == xtype) return go(x);
    return go((float*)nullptr);
  });
}

bool bad_sizes(int64_t outer, int64_t steps, int64_t inner) {
  return outer < 0 || steps < 0 || inner < 0 || inner > (1LL << 40) || outer > (1LL << 40) || steps > (1LL << 40);
}

void lay_args(Kargs& k, const Lay& l) {
  k.chunk_steps = l.steps;
  k.chunks = l.chunks;
  k.splits = l.splits;
}

}  // namespace

extern "C" int sb_gated_scan_plan(int64_t outer, int64_t steps, int64_t inner, int xtype, int64_t* chunks, int64_t* fwd_scratch,
                                  int64_t* bwd_scratch) {
  if (bad_sizes(outer, steps, inner) || xtype < SB_F32 || xtype > SB_F16 || !chunks || !fwd_scratch || !bwd_scratch) return -1001;
  *chunks = *fwd_scratch = *bwd_scratch = 0;
  if (outer == 0 || steps == 0 || inner == 0) return 0;
  const Lay l = lay_of(outer, steps, inner);
  *chunks = l.chunks;
  *fwd_scratch = *bwd_scratch = l.splits > 1 ? pairs_floats(l.splits, outer * inner) : 0;
  return 0;
}

extern "C" int sb_gated_scan_fwd(const sb_gated_scan_args* ap, void* stream) {
  if (!ap) return -1001;
  const sb_gated_scan_args& a = *ap;
  if (bad_sizes(a.outer, a.steps, a.inner) || a.so_x < 0 || a.st_x < 0 || a.so_g < 0 || a.st_g < 0) return -1004;
  if (a.outer == 0 || a.steps == 0 || a.inner == 0) return 0;
  if (!a.x || !a.gate || !a.h || !a.h_last) return -1005;
  return with_types(a.xtype, a.gtype, a.form, [&](auto* xt, auto* gt, auto form) -> int {
    using T = std::remove_pointer_t<decltype(xt)>;
    using G = std::remove_pointer_t<decltype(gt)>;
    const Lay l = lay_of(a.outer, a.steps, a.inner);
    if (l.tiles > 0x7fffffffLL) return -1006;
    if (l.splits > 1 && !a.scratch) return -1007;
    Kargs k = {};
    k.outer = a.outer; k.steps = a.steps; k.inner = a.inner; k.reverse = a.reverse != 0;
    k.x = a.x; k.so_x = a.so_x; k.st_x = a.st_x;
    k.gate = a.gate; k.so_g = a.so_g; k.st_g = a.st_g;
    k.h0 = a.h0; k.len = a.len; k.h = a.h; k.h_last = a.h_last; k.states = a.states; k.agg = a.scratch;
    lay_args(k, l);
    const dim3 block(64 * l.nw);
    const unsigned lds = l.nw > 1 ? 16 * 64 * l.nw : 0;
    if (l.splits > 1)
      hipLaunchKernelGGL((gated_scan_pair_kernel<T, G, form.value, true>), dim3((unsigned)l.tiles, l.splits - 1), block, lds, (hipStream_t)stream, k);
    hipLaunchKernelGGL((gated_scan_fwd_kernel<T, G, form.value>), dim3((unsigned)l.tiles, l.splits), block, lds, (hipStream_t)stream, k);
    SB_CHECK_LAUNCH();
    return 0;
  });
}

extern "C" int sb_gated_scan_bwd(const sb_gated_scan_bwd_args* ap, void* stream) {
  if (!ap) return -1001;
  const sb_gated_scan_bwd_args& a = *ap;
  if (bad_sizes(a.outer, a.steps, a.inner) || a.so_x < 0 || a.st_x < 0 || a.so_g < 0 || a.st_g < 0 || a.so_d < 0 || a.st_d < 0) return -1004;
  if (a.outer == 0 || a.steps == 0 || a.inner == 0) return 0;
  if (!a.x || !a.gate || !a.states || !a.dx || !a.dgate) return -1005;
  return with_types(a.xtype, a.gtype, a.form, [&](auto* xt, auto* gt, auto form) -> int {
    using T = std::remove_pointer_t<decltype(xt)>;
    using G = std::remove_pointer_t<decltype(gt)>;
    const Lay l = lay_of(a.outer, a.steps, a.inner);
    if (l.tiles > 0x7fffffffLL) return -1006;
    if (l.splits > 1 && !a.scratch) return -1007;
    Kargs k = {};
    k.outer = a.outer; k.steps = a.steps; k.inner = a.inner; k.reverse = a.reverse != 0;
    k.x = a.x; k.so_x = a.so_x; k.st_x = a.st_x;
    k.gate = a.gate; k.so_g = a.so_g; k.st_g = a.st_g;
    k.dh = a.dh; k.so_d = a.so_d; k.st_d = a.st_d;
    k.dlast = a.dlast; k.len = a.len; k.states = const_cast<float*>(a.states); k.agg = a.scratch;
    k.dx = a.dx; k.dgate = a.dgate; k.dh0 = a.dh0;
    lay_args(k, l);
    const dim3 block(64 * l.nw);
    const unsigned lds = l.nw > 1 ? 32 * 64 * l.nw : 0;
    if (l.splits > 1)
      hipLaunchKernelGGL((gated_scan_pair_kernel<T, G, form.value, false>), dim3((unsigned)l.tiles, l.splits - 1), block, lds, (hipStream_t)stream, k);
    hipLaunchKernelGGL((gated_scan_bwd_kernel<T, G, form.value>), dim3((unsigned)l.tiles, l.splits), block, lds, (hipStream_t)stream, k);
    SB_CHECK_LAUNCH();
    return 0;
  });
}

extern "C" int sb_gated_scan_step(const void* x, const void* gate, float* state, void* y, int64_t rows, int64_t inner, int64_t ld_x,
                                  int64_t ld_g, int xtype, int gtype, int form, void* stream) {
  if (bad_sizes(rows, 1, inner) || ld_x < 0 || ld_g < 0) return -1004;
  if (rows == 0 || inner == 0) return 0;
  if (!x || !gate || !state || !y) return -1005;
  return with_types(xtype, gtype, form, [&](auto* xt, auto* gt, auto f) -> int {
    using T = std::remove_pointer_t<decltype(xt)>;
    using G = std::remove_pointer_t<decltype(gt)>;
    const int64_t per_row = (inner + 3) / 4, total = rows * per_row, grid = (total + 255) / 256;
    if (grid > 0x7fffffffLL) return -1006;
    hipLaunchKernelGGL((gated_scan_step_kernel<T, G, f.value>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, (const T*)x,
                       (const G*)gate, state, (T*)y, inner, ld_x, ld_g, per_row, total);
    SB_CHECK_LAUNCH();
    return 0;
  });
}
