// Gated linear recurrence over the middle axis of [outer, steps, inner]:  h_t = a_t h_{t-1} + b_t, forward, backward, one step.
//
// Steps are joined as pairs (A, B): h -> A h + B; (A2, B2) after (A1, B1) is (A2 A1, A2 B1 + B2).  A thread holds V channels of S
// consecutive steps in registers and joins them in order; the threads along time are joined over lanes (distances 1, 2, 4, ...),
// waves through LDS, and the state is carried from chunk to chunk by the same workgroup, so x and gate are read once and the
// order of all products is fixed by the sizes.  Where there are too few columns (sequence x channel tile) to fill the chip, time is
// cut into segments: a first kernel makes each segment's pair, the second joins those in front of its own.
// Steps that a sequence does not have (behind its length, behind the last chunk) are (1, 0) by selection, whatever memory holds.
//
// The backward pass makes h_{t-1} again in fp32 from the states the forward pass left in front of every chunk, and walks
//   G_t = dh_t + c_{t+1},  c_t = a_t G_t
// down the same chunks: the pairs are (A, D): c -> A c + D, with A the forward pass's product.
#include "sb_seq_common.h"

namespace {

constexpr int S = 8;               // steps a thread holds
constexpr int kMaxSplits = 64;

// how a wave is laid over a column: lane = (column of the wave, segment, channel vector)
struct Lay {
  int lc, lseg, nw;                // lanes along channels, lanes along time, waves along time (powers of two)
  int64_t tiles, cols;             // channel tiles of a sequence, columns
  int per;                         // columns of a workgroup
  int64_t steps;                   // steps of a chunk
  int64_t groups() const { return (cols + per - 1) / per; }
};

int pow2_up(int64_t v, int most) {
  int p = 1;
  while (p < most && p < v) p *= 2;
  return p;
}

Lay lay_of(int64_t outer, int64_t steps, int64_t inner, int V, int full_lc) {
  Lay l;
  l.lc = pow2_up((inner + V - 1) / V, full_lc);
  l.lseg = pow2_up((steps + S - 1) / S, 64 / l.lc);
  l.tiles = (inner + l.lc * V - 1) / (l.lc * V);
  l.cols = outer * l.tiles;
  l.per = 64 / (l.lc * l.lseg);
  l.nw = l.per == 1 && steps > (int64_t)l.lseg * S && l.cols < 2048 ? 4 : 1;
  l.steps = (int64_t)l.lseg * l.nw * S;
  return l;
}

// channels of a thread and lanes along channels: 128 bytes of a step's row
int fwd_vec(int64_t inner, int xtype) { return xtype == SB_F32 ? (inner < 4 ? 1 : 4) : (inner < 8 ? 1 : 8); }
int bwd_vec(int64_t inner) { return inner < 4 ? 1 : 4; }
Lay fwd_lay(int64_t outer, int64_t steps, int64_t inner, int xtype) { return lay_of(outer, steps, inner, fwd_vec(inner, xtype), 8); }
Lay bwd_lay(int64_t outer, int64_t steps, int64_t inner, int xtype) { return lay_of(outer, steps, inner, bwd_vec(inner), xtype == SB_F32 ? 8 : 16); }

int splits_of(const Lay& l, int64_t steps) {
  const int64_t chunks = (steps + l.steps - 1) / l.steps, waves = l.groups() * l.nw;
  if (waves >= 1024 || chunks < 4) return 1;
  return (int)std::min<int64_t>(std::min<int64_t>(kMaxSplits, chunks / 2), (2048 + waves - 1) / waves);
}

struct Kargs {
  int64_t outer, steps, inner, tiles, cols, keep;      // keep: steps between two kept states
  int lc, lseg, reverse, splits;
  int64_t chunks, chunk_steps;
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

// Where a thread stands.  A sequence whose channels do not fill its last tile's vectors has that tile's vectors moved back to end
// with the last channel: two threads then make the same channels, to the same bits, and no vector is cut (V = 1 where inner < V).
template <int V> struct Place {
  int lane, wave, lc, seg, tseg;
  bool on;                                // the thread has channels
  int64_t o, c, lo, hi;                   // sequence, first channel, live steps [lo, hi) in the order of the walk
  bool all;                               // every thread of the workgroup has
  SB_DEVINL Place(const Kargs& k) {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    lc = lane & (k.lc - 1);
    seg = (lane / k.lc) & (k.lseg - 1);
    tseg = wave * k.lseg + seg;
    const int per = 64 / (k.lc * k.lseg);
    const int64_t col = (int64_t)blockIdx.x * per + lane / (k.lc * k.lseg);
    o = col / k.tiles;
    c = (col - o * k.tiles) * (k.lc * V) + lc * V;
    on = col < k.cols && c < k.inner;
    int64_t n = 0;
    if (on) {
      c = min(c, k.inner - V);
      n = k.len ? min(max(k.len[o], (int64_t)0), k.steps) : k.steps;
    } else {
      o = c = 0;
    }
    lo = k.reverse ? k.steps - n : 0;
    hi = k.reverse ? k.steps : n;
    all = __syncthreads_and(on) != 0;
  }
  // live steps of the thread's S from `first` on, as a bit each
  SB_DEVINL unsigned live(int64_t first) const {
    const int n0 = (int)min(max(lo - first, (int64_t)0), (int64_t)S), n1 = (int)min(max(hi - first, (int64_t)0), (int64_t)S);
    return ((1u << n1) - 1u) & ~((1u << n0) - 1u);
  }
};

template <class E, int V> SB_DEVINL void load_steps(Vec<E, V> (&v)[S], const void* base, int64_t so, int64_t st, const Place<V>& p, const Kargs& k,
                                                    int64_t t0, bool full) {
  const int64_t first = t0 + (int64_t)p.tseg * S;
  const int64_t step = k.reverse ? -st : st;
  const E* at = (const E*)base + p.o * so + p.c + (k.reverse ? k.steps - 1 - first : first) * st;
  if (full) {
#pragma unroll
    for (int s = 0; s < S; ++s) v[s] = vload<E, V>(at + s * step);
  } else {
    const unsigned live = p.live(first);
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[s].v[i] = (E)0.f;
      if (live >> s & 1) v[s] = vload<E, V>(at + s * step);
    }
  }
}

template <class E, int V> SB_DEVINL void store_steps(void* base, const Vec<E, V> (&v)[S], const Place<V>& p, const Kargs& k, int64_t t0, bool full) {
  const int64_t first = t0 + (int64_t)p.tseg * S;
  const int64_t step = k.reverse ? -k.inner : k.inner;
  E* at = (E*)base + (p.o * k.steps + (k.reverse ? k.steps - 1 - first : first)) * k.inner + p.c;
  if (full) {
#pragma unroll
    for (int s = 0; s < S; ++s) vstore<E, V>(at + s * step, v[s]);
  } else if (p.on) {
    const int n = (int)min(max(k.steps - first, (int64_t)0), (int64_t)S);
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (s < n) vstore<E, V>(at + s * step, v[s]);
  }
}

// lanes' pairs, in place, to the pair of all segments in front of (UP) / behind (!UP) the thread's own within its wave; -> the wave's whole in tot
template <bool UP, int V> SB_DEVINL void join_lanes(float (&A)[V], float (&B)[V], const Place<V>& p, const Kargs& k, float (&tA)[V], float (&tB)[V]) {
  for (int d = 1; d < k.lseg; d *= 2) {
    const int from = UP ? p.lane - d * k.lc : p.lane + d * k.lc;
    const bool has = UP ? p.seg >= d : p.seg + d < k.lseg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = __shfl(A[i], from & 63, 64), b = __shfl(B[i], from & 63, 64);
      if (has) {
        B[i] = __builtin_fmaf(A[i], b, B[i]);
        A[i] *= a;
      }
    }
  }
  const int base = p.lane - p.seg * k.lc;
  const int end = UP ? base + (k.lseg - 1) * k.lc : base, from = UP ? p.lane - k.lc : p.lane + k.lc;
  const bool has = UP ? p.seg > 0 : p.seg < k.lseg - 1;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    tA[i] = __shfl(A[i], end, 64);
    tB[i] = __shfl(B[i], end, 64);
    const float a = __shfl(A[i], from & 63, 64), b = __shfl(B[i], from & 63, 64);
    A[i] = has ? a : 1.f;
    B[i] = has ? b : 0.f;
  }
}

// carry over the waves: `in` = what enters the thread's wave, `carry` = what leaves the workgroup's chunk
template <bool UP, int V, int NW> SB_DEVINL void join_waves(float (*lds)[16 * V][2], const float (&tA)[V], const float (&tB)[V], const Place<V>& p,
                                                            float (&carry)[V], float (&in)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) in[i] = carry[i];
  if constexpr (NW == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = __builtin_fmaf(tA[i], carry[i], tB[i]);
  } else {
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int j = UP ? w : NW - 1 - w;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (j == p.wave) in[i] = carry[i];
        carry[i] = __builtin_fmaf(lds[j][p.lc * V + i][0], carry[i], lds[j][p.lc * V + i][1]);
      }
    }
  }
}
template <int V> SB_DEVINL void put_waves(float (*lds)[16 * V][2], const float (&tA)[V], const float (&tB)[V], const Place<V>& p) {
  if (p.seg == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lds[p.wave][p.lc * V + i][0] = tA[i];
      lds[p.wave][p.lc * V + i][1] = tB[i];
    }
  }
}

template <class G, int FORM, int V> SB_DEVINL void coefficients(const Vec<G, V>& g, float (&a)[V], float (&one_less)[V], bool live) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (FORM == SB_SCAN_SIGMOID)
      logistic((float)g.v[i], a[i], one_less[i]);
    else {
      a[i] = (float)g.v[i];
      one_less[i] = 1.f;
    }
    if (!live) {
      a[i] = 1.f;
      one_less[i] = 0.f;
    }
  }
}

// state in front of split `split`: h0 and the pairs of the earlier ones (UP), dlast and those of the later ones (!UP)
template <bool UP, int V> SB_DEVINL void fold_splits(float (&carry)[V], const float* start, const Place<V>& p, const Kargs& k, int split) {
  const int64_t oc = p.o * k.inner + p.c, plane = k.outer * k.inner;
#pragma unroll
  for (int i = 0; i < V; ++i) carry[i] = 0.f;
  if (!p.on) return;
  if (start) {
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = start[oc + i];
  }
  for (int j = UP ? 0 : k.splits - 1; UP ? j < split : j > split; j += UP ? 1 : -1) {
    const Vec<float, V> A = vload<float, V>(k.agg + (2 * j) * plane + oc), B = vload<float, V>(k.agg + (2 * j + 1) * plane + oc);
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = __builtin_fmaf(A.v[i], carry[i], B.v[i]);
  }
}

// MODE 0: h, states, h_last.  MODE 1: the pair of segment blockIdx.y into agg.
template <class T, class G, int FORM, int V, int NW, int MODE>
__global__ __launch_bounds__(64 * NW) void gated_scan_fwd_kernel(Kargs k) {
  __shared__ float lds[2][NW][16 * V][2];
  const Place<V> p(k);
  const int split = blockIdx.y;
  const int64_t c0 = k.chunks * split / k.splits, c1 = k.chunks * (split + 1) / k.splits;
  float carry[V], whole[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    carry[i] = 0.f;
    whole[i] = 1.f;
  }
  if constexpr (MODE == 0) fold_splits<true, V>(carry, k.h0, p, k, split);
  Vec<T, V> x[S];
  Vec<G, V> g[S];
  const auto is_full = [&](int64_t chunk) {
    const int64_t t0 = chunk * k.chunk_steps;
    return p.all && !k.len && t0 + k.chunk_steps <= k.steps;
  };
  load_steps<T, V>(x, k.x, k.so_x, k.st_x, p, k, c0 * k.chunk_steps, is_full(c0));
  load_steps<G, V>(g, k.gate, k.so_g, k.st_g, p, k, c0 * k.chunk_steps, is_full(c0));
  for (int64_t ch = c0; ch < c1; ++ch) {
    const int64_t t0 = ch * k.chunk_steps, first = t0 + (int64_t)p.tseg * S;
    const bool full = is_full(ch);
    const unsigned live = p.live(first);
    float a[S][V], b[S][V], A[V], B[V];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      coefficients<G, FORM, V>(g[s], a[s], b[s], full || (live >> s & 1));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        b[s][i] *= (float)x[s].v[i];
        A[i] = s ? A[i] * a[s][i] : a[s][i];
        B[i] = s ? __builtin_fmaf(a[s][i], B[i], b[s][i]) : b[s][i];
      }
    }
    if (ch + 1 < c1) {
      load_steps<T, V>(x, k.x, k.so_x, k.st_x, p, k, t0 + k.chunk_steps, is_full(ch + 1));
      load_steps<G, V>(g, k.gate, k.so_g, k.st_g, p, k, t0 + k.chunk_steps, is_full(ch + 1));
    }
    float tA[V], tB[V], in[V];
    join_lanes<true, V>(A, B, p, k, tA, tB);
    if constexpr (NW > 1) {
      put_waves<V>(lds[ch & 1], tA, tB, p);
      __syncthreads();
    }
    if constexpr (MODE == 1) {
      if constexpr (NW == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) whole[i] *= tA[i];
      } else {
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int i = 0; i < V; ++i) whole[i] *= lds[ch & 1][w][p.lc * V + i][0];
      }
    }
    join_waves<true, V, NW>(lds[ch & 1], tA, tB, p, carry, in);
    if constexpr (MODE == 0) {
      float h[V];
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = __builtin_fmaf(A[i], in[i], B[i]);
      if (k.states && p.on && (first & (k.keep - 1)) == 0 && first < k.steps) {
        Vec<float, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = h[i];
        vstore<float, V>(k.states + (first / k.keep) * (k.outer * k.inner) + p.o * k.inner + p.c, o);
      }
      Vec<T, V> out[S];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const bool lives = full || (live >> s & 1);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[i] = __builtin_fmaf(a[s][i], h[i], b[s][i]);
          out[s].v[i] = lives ? (T)h[i] : (T)0.f;
        }
      }
      store_steps<T, V>(k.h, out, p, k, t0, full);
    }
  }
  if (p.tseg == 0 && p.on) {
    const int64_t oc = p.o * k.inner + p.c;
    Vec<float, V> o, w;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o.v[i] = carry[i];
      w.v[i] = whole[i];
    }
    if constexpr (MODE == 0) {
      if (split == k.splits - 1) vstore<float, V>(k.h_last + oc, o);
    } else {
      const int64_t plane = k.outer * k.inner;
      vstore<float, V>(k.agg + (2 * split) * plane + oc, w);
      vstore<float, V>(k.agg + (2 * split + 1) * plane + oc, o);
    }
  }
}

// MODE 0: dx, dgate, dh0.  MODE 1: the pair (A, D) of segment blockIdx.y + 1 into agg.
template <class T, class G, int FORM, int V, int NW, int MODE>
__global__ __launch_bounds__(64 * NW) void gated_scan_bwd_kernel(Kargs k) {
  __shared__ float lds[2][2][NW][16 * V][2];
  const Place<V> p(k);
  const int split = blockIdx.y + (MODE == 1 ? 1 : 0);
  const int64_t c0 = k.chunks * split / k.splits, c1 = k.chunks * (split + 1) / k.splits;
  const int64_t oc = p.o * k.inner + p.c, plane = k.outer * k.inner;
  float carry[V], whole[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    carry[i] = 0.f;
    whole[i] = 1.f;
  }
  if constexpr (MODE == 0) fold_splits<false, V>(carry, k.dlast, p, k, split);
  Vec<T, V> x[S], d[S];
  Vec<G, V> g[S];
  Vec<float, V> state;
  const auto is_full = [&](int64_t chunk) {
    const int64_t t0 = chunk * k.chunk_steps;
    return p.all && !k.len && t0 + k.chunk_steps <= k.steps;
  };
  const auto load = [&](int64_t ch) __attribute__((always_inline)) {
    const int64_t t0 = ch * k.chunk_steps;
    const bool full = is_full(ch);
    load_steps<G, V>(g, k.gate, k.so_g, k.st_g, p, k, t0, full);
    if (k.dh) load_steps<T, V>(d, k.dh, k.so_d, k.st_d, p, k, t0, full);
    if constexpr (MODE == 0) {
      load_steps<T, V>(x, k.x, k.so_x, k.st_x, p, k, t0, full);
      if (p.on) state = vload<float, V>(k.states + ch * plane + oc);
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < V; ++i) d[s].v[i] = (T)0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) state.v[i] = 0.f;
  load(c1 - 1);
  for (int64_t ch = c1 - 1; ch >= c0; --ch) {
    const int64_t t0 = ch * k.chunk_steps, first = t0 + (int64_t)p.tseg * S;
    const bool full = is_full(ch);
    const unsigned live = p.live(first);
    float a[S][V], ol[S][V], A[V], D[V];
    float xf[S][V], df[S][V];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const bool lives = full || (live >> s & 1);
      coefficients<G, FORM, V>(g[s], a[s], ol[s], lives);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xf[s][i] = MODE == 0 ? (float)x[s].v[i] : 0.f;      // (dead steps were loaded as 0)
        df[s][i] = (float)d[s].v[i];
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        A[i] = s < S - 1 ? A[i] * a[s][i] : a[s][i];
        D[i] = a[s][i] * (s < S - 1 ? df[s][i] + D[i] : df[s][i]);
      }
    float fA[V], fB[V], fin[V];
    if constexpr (MODE == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        fA[i] = A[i];
        fB[i] = ol[0][i] * xf[0][i];
      }
#pragma unroll
      for (int s = 1; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) fB[i] = __builtin_fmaf(a[s][i], fB[i], ol[s][i] * xf[s][i]);
#pragma unroll
      for (int i = 0; i < V; ++i) fin[i] = state.v[i];
    }
    if (ch > c0) load(ch - 1);
    float tA[V], tD[V], in[V];
    join_lanes<false, V>(A, D, p, k, tA, tD);
    if constexpr (NW > 1) put_waves<V>(lds[ch & 1][0], tA, tD, p);
    if constexpr (MODE == 0) {
      float ftA[V], ftB[V], hin[V];
      join_lanes<true, V>(fA, fB, p, k, ftA, ftB);
      if constexpr (NW > 1) {
        put_waves<V>(lds[ch & 1][1], ftA, ftB, p);
        __syncthreads();
      }
      join_waves<false, V, NW>(lds[ch & 1][0], tA, tD, p, carry, in);
      join_waves<true, V, NW>(lds[ch & 1][1], ftA, ftB, p, fin, hin);
      float hb[S][V];
#pragma unroll
      for (int i = 0; i < V; ++i) hb[0][i] = __builtin_fmaf(fA[i], hin[i], fB[i]);
#pragma unroll
      for (int s = 1; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) hb[s][i] = __builtin_fmaf(a[s - 1][i], hb[s - 1][i], ol[s - 1][i] * xf[s - 1][i]);
      float c[V];
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = __builtin_fmaf(A[i], in[i], D[i]);
      Vec<T, V> dx[S];
      Vec<G, V> dg[S];
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        const bool lives = full || (live >> s & 1);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float gt = df[s][i] + c[i];
          c[i] = a[s][i] * gt;
          float vx, vg;
          if constexpr (FORM == SB_SCAN_SIGMOID) {
            vx = ol[s][i] * gt;
            vg = gt * (hb[s][i] - xf[s][i]) * (a[s][i] * ol[s][i]);
          } else {
            vx = gt;
            vg = gt * hb[s][i];
          }
          dx[s].v[i] = lives ? (T)vx : (T)0.f;
          dg[s].v[i] = lives ? (G)vg : (G)0.f;
        }
      }
      store_steps<T, V>(k.dx, dx, p, k, t0, full);
      store_steps<G, V>(k.dgate, dg, p, k, t0, full);
    } else {
      if constexpr (NW > 1) {
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int i = 0; i < V; ++i) whole[i] *= lds[ch & 1][0][w][p.lc * V + i][0];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) whole[i] *= tA[i];
      }
      join_waves<false, V, NW>(lds[ch & 1][0], tA, tD, p, carry, in);
    }
  }
  if (p.tseg == 0 && p.on) {
    Vec<float, V> o, w;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o.v[i] = carry[i];
      w.v[i] = whole[i];
    }
    if constexpr (MODE == 0) {
      if (split == 0 && k.dh0) vstore<float, V>(k.dh0 + oc, o);
    } else {
      vstore<float, V>(k.agg + (2 * split) * plane + oc, w);
      vstore<float, V>(k.agg + (2 * split + 1) * plane + oc, o);
    }
  }
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
  coefficients<G, FORM, V>(gv, a, b, true);
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

void lay_args(Kargs& k, const Lay& l, int splits, int64_t keep) {
  k.tiles = l.tiles;
  k.cols = l.cols;
  k.lc = l.lc;
  k.lseg = l.lseg;
  k.chunk_steps = l.steps;
  k.chunks = (k.steps + l.steps - 1) / l.steps;
  k.splits = splits;
  k.keep = keep;
}

}  // namespace

extern "C" int sb_gated_scan_plan(int64_t outer, int64_t steps, int64_t inner, int xtype, int64_t* chunks, int64_t* fwd_scratch,
                                  int64_t* bwd_scratch) {
  if (bad_sizes(outer, steps, inner) || xtype < SB_F32 || xtype > SB_F16 || !chunks || !fwd_scratch || !bwd_scratch) return -1001;
  *chunks = *fwd_scratch = *bwd_scratch = 0;
  if (outer == 0 || steps == 0 || inner == 0) return 0;
  const Lay f = fwd_lay(outer, steps, inner, xtype), b = bwd_lay(outer, steps, inner, xtype);
  *chunks = (steps + b.steps - 1) / b.steps;
  const int sf = splits_of(f, steps), sb = splits_of(b, steps);
  *fwd_scratch = sf > 1 ? 2 * sf * outer * inner : 0;
  *bwd_scratch = sb > 1 ? 2 * sb * outer * inner : 0;
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
    const Lay l = fwd_lay(a.outer, a.steps, a.inner, a.xtype);
    const int splits = splits_of(l, a.steps);
    if (l.groups() > 0x7fffffffLL) return -1006;
    if (splits > 1 && !a.scratch) return -1007;
    Kargs k = {};
    k.outer = a.outer; k.steps = a.steps; k.inner = a.inner; k.reverse = a.reverse != 0;
    k.x = a.x; k.so_x = a.so_x; k.st_x = a.st_x;
    k.gate = a.gate; k.so_g = a.so_g; k.st_g = a.st_g;
    k.h0 = a.h0; k.len = a.len; k.h = a.h; k.h_last = a.h_last; k.states = a.states; k.agg = a.scratch;
    lay_args(k, l, splits, bwd_lay(a.outer, a.steps, a.inner, a.xtype).steps);
    const auto go = [&](auto v, auto nw) {
      constexpr int V = decltype(v)::value, NW = decltype(nw)::value;
      if (splits > 1)
        hipLaunchKernelGGL((gated_scan_fwd_kernel<T, G, form.value, V, NW, 1>), dim3((unsigned)l.groups(), splits - 1), dim3(64 * NW), 0, (hipStream_t)stream, k);
      hipLaunchKernelGGL((gated_scan_fwd_kernel<T, G, form.value, V, NW, 0>), dim3((unsigned)l.groups(), splits), dim3(64 * NW), 0, (hipStream_t)stream, k);
    };
    const auto waves = [&](auto v) {
      if (l.nw == 4) go(v, std::integral_constant<int, 4>()); else go(v, std::integral_constant<int, 1>());
    };
    if (fwd_vec(a.inner, a.xtype) == 1) waves(std::integral_constant<int, 1>()); else waves(std::integral_constant<int, vec_of<T>()>());
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
    const Lay l = bwd_lay(a.outer, a.steps, a.inner, a.xtype);
    const int splits = splits_of(l, a.steps);
    if (l.groups() > 0x7fffffffLL) return -1006;
    if (splits > 1 && !a.scratch) return -1007;
    Kargs k = {};
    k.outer = a.outer; k.steps = a.steps; k.inner = a.inner; k.reverse = a.reverse != 0;
    k.x = a.x; k.so_x = a.so_x; k.st_x = a.st_x;
    k.gate = a.gate; k.so_g = a.so_g; k.st_g = a.st_g;
    k.dh = a.dh; k.so_d = a.so_d; k.st_d = a.st_d;
    k.dlast = a.dlast; k.len = a.len; k.states = const_cast<float*>(a.states); k.agg = a.scratch;
    k.dx = a.dx; k.dgate = a.dgate; k.dh0 = a.dh0;
    lay_args(k, l, splits, l.steps);
    const auto go = [&](auto v, auto nw) {
      constexpr int V = decltype(v)::value, NW = decltype(nw)::value;
      if (splits > 1)
        hipLaunchKernelGGL((gated_scan_bwd_kernel<T, G, form.value, V, NW, 1>), dim3((unsigned)l.groups(), splits - 1), dim3(64 * NW), 0, (hipStream_t)stream, k);
      hipLaunchKernelGGL((gated_scan_bwd_kernel<T, G, form.value, V, NW, 0>), dim3((unsigned)l.groups(), splits), dim3(64 * NW), 0, (hipStream_t)stream, k);
    };
    const auto waves = [&](auto v) {
      if (l.nw == 4) go(v, std::integral_constant<int, 4>()); else go(v, std::integral_constant<int, 1>());
    };
    if (bwd_vec(a.inner) == 1) waves(std::integral_constant<int, 1>()); else waves(std::integral_constant<int, 4>());
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
