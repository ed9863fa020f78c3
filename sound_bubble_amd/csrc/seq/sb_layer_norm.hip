// Layer norm over the last axis, forward and backward, any width.
//
// A row belongs to a group of L lanes (a part of a wave, a wave, or a workgroup), each holding K vectors of 16 bytes of it in
// registers, so x is read once; the mean goes first and the squares are those of x - mean, in fp32.  Groups walk over rows
// with a stride, which keeps w and b -- and in the backward pass the sums of dw and db -- in registers, and the next row's loads are under
// way while a row is worked on.  Every load is a whole vector: those that would pass the row's end are moved back to end with it, and what
// they hold twice (all of it, where a lane has nothing) counts once.
#include "sb_seq_common.h"

namespace {

// sum over the group; a group larger than a wave goes through LDS (two buffers in turn: one barrier a sum)
template <int L> struct Group {
  float* lds;
  int turn = 0;
  SB_DEVINL float sum(float v) {
    if constexpr (L <= 64) return lane_sum<L>(v);
    constexpr int W = L / 64;
    v = lane_sum<64>(v);
    float* at = lds + turn * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += at[w];
    return s;
  }
  SB_DEVINL void sum2(float& a, float& b) {
    if constexpr (L <= 64) {
      a = lane_sum<L>(a);
      b = lane_sum<L>(b);
    } else {
      constexpr int W = L / 64;
      a = lane_sum<64>(a);
      b = lane_sum<64>(b);
      float* at = lds + turn * 2 * W;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
        at[threadIdx.x >> 6] = a;
        at[W + (threadIdx.x >> 6)] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        a += at[w];
        b += at[W + w];
      }
    }
  }
};

template <int L> constexpr int threads_of() { return L > 256 ? L : 256; }

// a lane's K vectors of a row of n >= V elements
template <int V, int L, int K> struct Cols {
  int lane, n;
  SB_DEVINL int at(int k) const { return min((k * L + lane) * V, n - V); }
  SB_DEVINL int twice(int k) const { return (k * L + lane) * V - (n - V); }      // elements in front that another lane has (<= 0: none, >= V: all)
  SB_DEVINL bool exact() const { return n == L * K * V; }
  template <class E> SB_DEVINL void load(Vec<E, V> (&v)[K], const E* row) const {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = vload<E, V>(row + at(k));
  }
  template <class E> SB_DEVINL void store(E* row, const Vec<E, V>& v, int k) const {
    const int d = twice(k);
    if (d <= 0) {
      vstore<E, V>(row + (k * L + lane) * V, v);
    } else if (d < V) {
#pragma unroll
      for (int i = 1; i < V; ++i)
        if (i >= d) row[n - V + i] = v.v[i];
    }
  }
};

template <class T, class W, int V, int L, int K>
__global__ __launch_bounds__(threads_of<L>()) void layer_norm_fwd_kernel(sb_layer_norm_args a) {
  constexpr int G = threads_of<L>() / L;
  __shared__ float lds[L > 64 ? 2 * (L / 64) : 1];
  Group<L> group{lds};
  const Cols<V, L, K> cols{(int)threadIdx.x % L, (int)a.n};
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L;
  if (row >= a.rows) return;      // (a group; a workgroup where that is one)
  constexpr bool kAhead = L < 1024 || K < 4;      // (the registers of a workgroup of 1024 do not hold another row)
  Vec<T, V> xv[K], next[K];
  if constexpr (kAhead) cols.load(next, (const T*)a.x + row * a.ldx);
  constexpr bool kLean = K == 8;      // (nor w and b, which the caches hold: fp32 3000 x 32768 218 -> 176 us)
  Vec<W, V> w[kLean ? 1 : K], b[kLean ? 1 : K];
  if constexpr (!kLean) {
    if (a.w) cols.load(w, (const W*)a.w);
    if (a.b) cols.load(b, (const W*)a.b);
  }
  const float rn = 1.f / (float)a.n;
  for (; row < a.rows; row += step) {
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < K; ++k) xv[k] = next[k];
      if (row + step < a.rows) cols.load(next, (const T*)a.x + (row + step) * a.ldx);
    } else {
      cols.load(xv, (const T*)a.x + row * a.ldx);
    }
    float s = 0.f;
    const auto sum = [&](auto whole) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s += whole.value || i >= cols.twice(k) ? (float)xv[k].v[i] : 0.f;
    };
    if (cols.exact()) sum(std::true_type()); else sum(std::false_type());
    const float mean = group.sum(s) * rn;
    s = 0.f;
    const auto squares = [&](auto whole) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = whole.value || i >= cols.twice(k) ? (float)xv[k].v[i] - mean : 0.f;
          s += d * d;
        }
    };
    if (cols.exact()) squares(std::true_type()); else squares(std::false_type());
    const float rstd = 1.f / sqrtf(group.sum(s) * rn + a.eps);
    T* y = (T*)a.y + row * a.n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      constexpr bool kHeld = !kLean;
      if constexpr (kLean) {
        if (a.w) w[0] = vload<W, V>((const W*)a.w + cols.at(k));
        if (a.b) b[0] = vload<W, V>((const W*)a.b + cols.at(k));
      }
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = ((float)xv[k].v[i] - mean) * rstd;
        if (a.w) v *= (float)w[kHeld ? k : 0].v[i];
        if (a.b) v += (float)b[kHeld ? k : 0].v[i];
        o.v[i] = (T)v;
      }
      cols.store(y, o, k);
    }
    if (cols.lane == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// rows wider than a workgroup's registers: three passes over the row, which the caches hold
template <class T, class W>
__global__ __launch_bounds__(1024) void layer_norm_fwd_wide_kernel(sb_layer_norm_args a) {
  constexpr int V = vec_of<T>(), L = 1024;
  __shared__ float lds[2 * (L / 64)];
  Group<L> group{lds};
  const float rn = 1.f / (float)a.n;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    T* y = (T*)a.y + row * a.n;
    float s = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.n; c += (int64_t)L * V) {
      const Vec<T, V> v = vload_n<T, V>(x + c, (int)min((int64_t)V, a.n - c));
#pragma unroll
      for (int i = 0; i < V; ++i) s += (float)v.v[i];
    }
    const float mean = group.sum(s) * rn;
    s = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.n; c += (int64_t)L * V) {
      const int m = (int)min((int64_t)V, a.n - c);
      const Vec<T, V> v = vload_n<T, V>(x + c, m);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = i < m ? (float)v.v[i] - mean : 0.f;
        s += d * d;
      }
    }
    const float rstd = 1.f / sqrtf(group.sum(s) * rn + a.eps);
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.n; c += (int64_t)L * V) {
      const int m = (int)min((int64_t)V, a.n - c);
      Vec<T, V> v = vload_n<T, V>(x + c, m);
      Vec<W, V> w, b;
      if (a.w) w = vload_n<W, V>((const W*)a.w + c, m);
      if (a.b) b = vload_n<W, V>((const W*)a.b + c, m);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float r = ((float)v.v[i] - mean) * rstd;
        if (a.w) r *= (float)w.v[i];
        if (a.b) r += (float)b.v[i];
        v.v[i] = (T)r;
      }
      vstore_n<T, V>(y + c, v, m);
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Whether a group's registers hold the sums of dw and db beside the rows; where not, a kernel of its own reads x and dy once more for them
// (bf16 16384 x 16384: 512 us, with the sums inside and spilled 705; fp32 3000 x 24000: 296, the wide kernel's two passes 365)
constexpr bool sums_inside(int L, int K, bool f32) { return L < 1024 || (f32 && K <= 4); }

// dx of every row, and (scratch given) a row of partial sums of dw and db a workgroup: scratch[(0 | 1)][workgroup][n]
template <class T, class W, int V, int L, int K>
__global__ __launch_bounds__(threads_of<L>()) void layer_norm_bwd_kernel(sb_layer_norm_bwd_args a) {
  constexpr int NT = threads_of<L>(), G = NT / L;
  __shared__ float lds[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float acc[G > 1 ? NT * V : 1];      // one vector a thread goes through it at a time
  Group<L> group{lds};
  const Cols<V, L, K> cols{(int)threadIdx.x % L, (int)a.n};
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L;
  constexpr bool kAhead = L < 1024 || K < 3;      // another row's loads ahead, where the registers hold it
  constexpr bool kSums = sums_inside(L, K, V == 4);
  Vec<T, V> xv[K], gv[K], nx[K], ng[K];
  float mean, rstd, nmean = 0.f, nrstd = 0.f;
  const auto load = [&](int64_t r) __attribute__((always_inline)) {
    cols.load(nx, (const T*)a.x + r * a.ldx);
    cols.load(ng, (const T*)a.dy + r * a.lddy);
    nmean = a.mean[r];
    nrstd = a.rstd[r];
  };
  if (kAhead && row < a.rows) load(row);
  Vec<W, V> w[K];
  if (a.w) cols.load(w, (const W*)a.w);
  float dw[kSums ? K : 1][V], db[kSums ? K : 1][V];
  if constexpr (kSums) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  }
  const float rn = 1.f / (float)a.n;
  for (; row < a.rows; row += step) {
    if constexpr (!kAhead) load(row);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xv[k] = nx[k];
      gv[k] = ng[k];
    }
    mean = nmean;
    rstd = nrstd;
    if (kAhead && row + step < a.rows) load(row + step);
    float s1 = 0.f, s2 = 0.f;
    const auto sums = [&](auto whole) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float xh = ((float)xv[k].v[i] - mean) * rstd, g = whole.value || i >= cols.twice(k) ? (float)gv[k].v[i] : 0.f;
          const float q = a.w ? g * (float)w[k].v[i] : g;
          s1 += q;
          s2 += q * xh;
          if constexpr (kSums) {
            dw[k][i] += g * xh;
            db[k][i] += g;
          }
        }
    };
    if (cols.exact()) sums(std::true_type()); else sums(std::false_type());
    group.sum2(s1, s2);
    s1 *= rn;
    s2 *= rn;
    T* dx = (T*)a.dx + row * a.n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = ((float)xv[k].v[i] - mean) * rstd;
        const float q = a.w ? (float)gv[k].v[i] * (float)w[k].v[i] : (float)gv[k].v[i];
        o.v[i] = (T)(rstd * (q - s1 - xh * s2));
      }
      cols.store(dx, o, k);
    }
  }
  if constexpr (!kSums) return;
  if (!a.scratch) return;
  float* out[2] = {a.scratch + (int64_t)blockIdx.x * a.n, a.scratch + ((int64_t)gridDim.x + blockIdx.x) * a.n};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (which ? !a.db : !a.dw) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Vec<float, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = which ? db[kSums ? k : 0][i] : dw[kSums ? k : 0][i];
      if constexpr (G > 1) {      // the groups' sum, by the first group
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) acc[threadIdx.x * V + i] = o.v[i];
        __syncthreads();
        if (threadIdx.x >= L) continue;
        for (int g = 1; g < G; ++g)
#pragma unroll
          for (int i = 0; i < V; ++i) o.v[i] += acc[(g * L + threadIdx.x) * V + i];
      }
      cols.store(out[which], o, k);
    }
  }
}

// rows wider than a workgroup's registers: dx only, two passes over the row
template <class T, class W>
__global__ __launch_bounds__(1024) void layer_norm_bwd_wide_kernel(sb_layer_norm_bwd_args a) {
  constexpr int V = vec_of<T>(), L = 1024;
  __shared__ float lds[4 * (L / 64)];
  Group<L> group{lds};
  const float rn = 1.f / (float)a.n;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* dy = (const T*)a.dy + row * a.lddy;
    T* dx = (T*)a.dx + row * a.n;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.n; c += (int64_t)L * V) {
      const int m = (int)min((int64_t)V, a.n - c);
      const Vec<T, V> xv = vload_n<T, V>(x + c, m), gv = vload_n<T, V>(dy + c, m);
      Vec<W, V> w;
      if (a.w) w = vload_n<W, V>((const W*)a.w + c, m);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = a.w ? (float)gv.v[i] * (float)w.v[i] : (float)gv.v[i];
        s1 += q;
        s2 += q * (((float)xv.v[i] - mean) * rstd);
      }
    }
    group.sum2(s1, s2);
    s1 *= rn;
    s2 *= rn;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.n; c += (int64_t)L * V) {
      const int m = (int)min((int64_t)V, a.n - c);
      const Vec<T, V> xv = vload_n<T, V>(x + c, m), gv = vload_n<T, V>(dy + c, m);
      Vec<W, V> w;
      if (a.w) w = vload_n<W, V>((const W*)a.w + c, m);
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = a.w ? (float)gv.v[i] * (float)w.v[i] : (float)gv.v[i];
        o.v[i] = (T)(rstd * (q - s1 - ((float)xv.v[i] - mean) * rstd * s2));
      }
      vstore_n<T, V>(dx + c, o, m);
    }
  }
}

// ... and the column sums of it: a thread owns a vector of columns, a workgroup a range of rows
template <class T>
__global__ __launch_bounds__(256) void layer_norm_cols_kernel(sb_layer_norm_bwd_args a, int parts) {
  constexpr int V = vec_of<T>();
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (c >= a.n) return;
  const int64_t at = min(c, a.n - V);      // (the last vector ends with the row: its first columns are made twice, to the same bits)
  const int64_t per = (a.rows + parts - 1) / parts, r0 = blockIdx.y * per, r1 = min(a.rows, r0 + per);
  Vec<float, V> dw, db;
#pragma unroll
  for (int i = 0; i < V; ++i) dw.v[i] = db.v[i] = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const Vec<T, V> g = vload<T, V>((const T*)a.dy + r * a.lddy + at), x = vload<T, V>((const T*)a.x + r * a.ldx + at);
    const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      dw.v[i] += (float)g.v[i] * (((float)x.v[i] - mean) * rstd);
      db.v[i] += (float)g.v[i];
    }
  }
  vstore<float, V>(a.scratch + (int64_t)blockIdx.y * a.n + at, dw);
  vstore<float, V>(a.scratch + ((int64_t)parts + blockIdx.y) * a.n + at, db);
}

// dw, db from the workgroups' rows: 1024 threads are 32 columns x 32 ranges of rows
template <class W>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* scratch, int parts, int64_t n, void* dw, void* db) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + col;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const float* in = scratch + (int64_t)blockIdx.y * parts * n;
  float s = 0.f;
  if (c < n) {
#pragma unroll 16
    for (int p = part; p < parts; p += 32) s += in[(int64_t)p * n + c];
  }
  lds[part][col] = s;
  __syncthreads();
  if (part == 0 && c < n) {
    s = 0.f;
#pragma unroll
    for (int p = 0; p < 32; ++p) s += lds[p][col];
    ((W*)out)[c] = (W)s;
  }
}

// The groups in use.  Measured, us: forward, bf16 16384 x 4096: a wave with 8 vectors a lane 71, a workgroup of 256 with 2 47; backward, bf16
// 16384 x 2048: a wave with 4 50, a workgroup with 1 44, 50000 x 1280: a wave with 3 89, a workgroup with 1 115.  The backward pass's K vectors
// of x, dy, w, two of sums and the next row's have to fit the registers: 128 a lane in a workgroup of 1024, 256 in one of 512 (fp16 2309 x
// 16384: 512 x 4 158, 1024 x 2 without the sums 81; fp16 3000 x 32768: 1024 x 4 317, the wide kernel 254; forward, fp16 3000 x 50000:
// 1024 x 8 590, the wide kernel 213).
constexpr bool taken(int L, int K, bool f32, bool backward) {
  if (L <= 64) return K <= (backward ? 3 : 4);
  if (!backward) return !(L == 1024 && (K == 2 || (!f32 && K > 4)));
  return f32 ? !(L == 512 && K == 4) : (L == 1024 ? K <= 3 : L == 512 ? K == 3 : true);
}
// waves of the forward pass, whose groups walk over the rows: 1.45 M x 32 fp32: 68 us, with 8192 waves 77, with 2048 84; fp16 2309 x 16384:
// 31, with 8192 36
constexpr int64_t kFwdWaves = 4096;
// elements of a vector: 16 bytes, or one where the row is shorter than that
int vec_for(int64_t n, int xtype) {
  const int vec = xtype == SB_F32 ? 4 : 8;
  return n < vec ? 1 : vec;
}
// the group that holds a row of n elements: L lanes with K vectors each; L = 0: none does
struct Shape { int L, K; };
Shape shape_of(int64_t n, int xtype, bool backward) {
  const int vec = vec_for(n, xtype);
  const int64_t vecs = (n + vec - 1) / vec;
  if (vecs <= 64) {
    int L = 1;
    while (L < vecs) L *= 2;
    return {L, 1};
  }
  for (const Shape s : {Shape{64, 2}, {64, 3}, {64, 4}, {256, 1}, {256, 2}, {256, 3}, {256, 4}, {512, 3}, {512, 4}, {1024, 2}, {1024, 3}, {1024, 4},
                        {1024, 6}, {1024, 8}})
    if ((int64_t)s.L * s.K >= vecs && taken(s.L, s.K, xtype == SB_F32, backward)) return s;
  return {0, 0};
}


// f(integral_constant<V>, integral_constant<L>, integral_constant<K>)
template <class T, bool BACKWARD, class F> int with_shape(int64_t n, Shape s, F&& f) {
  constexpr std::integral_constant<int, vec_of<T>()> vec;
  constexpr std::integral_constant<int, 1> one;
  if (n < vec.value) {      // L >= n lanes of one element
    if (s.L == 1) return f(one, one, one);
    if (s.L == 2) return f(one, std::integral_constant<int, 2>(), one);
    if (s.L == 4) return f(one, std::integral_constant<int, 4>(), one);
    return f(one, std::integral_constant<int, 8>(), one);
  }
#define SB_CASE(l, k) \
  if constexpr (taken(l, k, std::is_same_v<T, float>, BACKWARD)) \
    if (s.L == l && s.K == k) return f(vec, std::integral_constant<int, l>(), std::integral_constant<int, k>());
  SB_CASE(1, 1) SB_CASE(2, 1) SB_CASE(4, 1) SB_CASE(8, 1) SB_CASE(16, 1) SB_CASE(32, 1) SB_CASE(64, 1) SB_CASE(64, 2) SB_CASE(64, 3) SB_CASE(64, 4)
  SB_CASE(256, 1) SB_CASE(256, 2) SB_CASE(256, 3) SB_CASE(256, 4) SB_CASE(512, 3) SB_CASE(512, 4)
  SB_CASE(1024, 2) SB_CASE(1024, 3) SB_CASE(1024, 4) SB_CASE(1024, 6) SB_CASE(1024, 8)
#undef SB_CASE
  return -1009;
}

// f(T*, W*)
template <class F> int with_types(int xtype, int wtype, F&& f) {
  return sb_with_type(xtype, [&](auto* x) -> int {
    if (wtype == xtype) return f(x, x);
    return f(x, (float*)nullptr);
  });
}

// Workgroups of the backward pass = rows of partial sums, each n floats of dw and db that are written and read once more: with few
// rows one a compute unit (fp16 2309 x 10007: 256 54 us, 512 77 us), with many two (bf16 16384 x 2048: 512 44 us, 256 50 us)
int64_t bwd_grid(int64_t rows, int64_t n, int xtype) {
  const Shape s = shape_of(n, xtype, true);
  if (!s.L || !sums_inside(s.L, s.K, xtype == SB_F32)) return std::min<int64_t>(rows, 128);      // (of the kernel for the sums alone)
  const int64_t per = s.L >= 256 ? 1 : 256 / s.L;
  return std::min<int64_t>((rows + per - 1) / per, s.L >= 256 && rows < 8192 ? 256 : 512);
}

}  // namespace

extern "C" int sb_layer_norm_fwd(const sb_layer_norm_args* ap, void* stream) {
  if (!ap) return -1001;
  const sb_layer_norm_args a = *ap;
  if (a.rows < 0 || a.n <= 0 || a.n > (1LL << 30) || a.ldx < 0 || (a.wtype != a.xtype && a.wtype != SB_F32)) return -1002;
  if (a.rows == 0) return 0;
  if (!a.x || !a.y || !a.mean != !a.rstd) return -1003;
  const Shape s = shape_of(a.n, a.xtype, false);
  return with_types(a.xtype, a.wtype, [&](auto* t, auto* wt) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(wt)>;
    if (!s.L) {
      hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<T, W>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(1024), 0, (hipStream_t)stream, a);
    } else {
      const int rc = with_shape<T, false>(a.n, s, [&](auto V, auto L, auto K) -> int {
        constexpr int per = threads_of<L.value>() / L.value;
        const int64_t grid = std::min<int64_t>((a.rows + per - 1) / per, kFwdWaves * 64 / threads_of<L.value>());
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W, V.value, L.value, K.value>), dim3((unsigned)grid), dim3(threads_of<L.value>()), 0, (hipStream_t)stream, a);
        return 0;
      });
      if (rc) return rc;
    }
    SB_CHECK_LAUNCH();
    return 0;
  });
}

extern "C" int64_t sb_layer_norm_bwd_scratch(int64_t rows, int64_t n, int xtype) { return rows <= 0 ? 0 : 2 * bwd_grid(rows, n, xtype) * n; }

extern "C" int sb_layer_norm_bwd(const sb_layer_norm_bwd_args* ap, void* stream) {
  if (!ap) return -1001;
  sb_layer_norm_bwd_args a = *ap;
  const bool sums = a.dw || a.db;
  if (a.rows < 0 || a.n <= 0 || a.n > (1LL << 30) || a.ldx < 0 || a.lddy < 0 || (a.wtype != a.xtype && a.wtype != SB_F32)) return -1002;
  if (a.rows > 0 && (!a.x || !a.dy || !a.dx || !a.mean || !a.rstd || (sums && !a.scratch))) return -1003;
  const Shape s = shape_of(a.n, a.xtype, true);
  const int grid = (int)bwd_grid(a.rows, a.n, a.xtype);
  return with_types(a.xtype, a.wtype, [&](auto* t, auto* wt) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(wt)>;
    const bool apart = a.rows > 0 && (!s.L || !sums_inside(s.L, s.K, std::is_same_v<T, float>));
    if (a.rows > 0 && !s.L) {
      hipLaunchKernelGGL((layer_norm_bwd_wide_kernel<T, W>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(1024), 0, (hipStream_t)stream, a);
    } else if (a.rows > 0) {
      if (!sums) a.scratch = nullptr;
      const int rc = with_shape<T, true>(a.n, s, [&](auto V, auto L, auto K) -> int {
        const int wgs = apart ? (int)std::min<int64_t>(a.rows, 512) : grid;
        hipLaunchKernelGGL((layer_norm_bwd_kernel<T, W, V.value, L.value, K.value>), dim3(wgs), dim3(threads_of<L.value>()), 0, (hipStream_t)stream, a);
        return 0;
      });
      if (rc) return rc;
    }
    SB_CHECK_LAUNCH();
    if (apart && sums) {
      hipLaunchKernelGGL((layer_norm_cols_kernel<T>), dim3((unsigned)((a.n / vec_of<T>() + 256) / 256), grid), dim3(256), 0, (hipStream_t)stream, a, grid);
      SB_CHECK_LAUNCH();
    }
    if (sums) {      // (no rows: no partial sums either, the sums are 0)
      hipLaunchKernelGGL((layer_norm_reduce_kernel<W>), dim3((unsigned)((a.n + 31) / 32), 2), dim3(1024), 0, (hipStream_t)stream, a.scratch,
                         a.rows > 0 ? grid : 0, a.n, a.dw, a.db);
      SB_CHECK_LAUNCH();
    }
    return 0;
  });
}
