// Layer norm over the last axis, forward and backward, any width.
//
// A row belongs to a group of L lanes (a part of a wave, a wave, or a workgroup), each holding K vectors of 16 bytes of it in
// registers, so x is read once; the mean goes first and the squares are those of x - mean, in fp32.  Groups walk over rows
// with a stride, which keeps w and b -- and in the backward pass the sums of dw and db -- in registers.
#include "sb_seq_common.h"

namespace {

constexpr int kMaxK = 8;

template <class T> SB_DEVINL float wload(const void* w, int wtype, int64_t i) {
  return wtype == SB_F32 ? ((const float*)w)[i] : (float)((const T*)w)[i];
}

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

template <class T, int L, int K>
__global__ __launch_bounds__(threads_of<L>()) void layer_norm_fwd_kernel(sb_layer_norm_args a) {
  constexpr int V = vec_of<T>(), G = threads_of<L>() / L;
  __shared__ float lds[L > 64 ? 2 * (L / 64) : 1];
  Group<L> group{lds};
  const int lane = threadIdx.x % L;
  const int n = (int)a.n;
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (k * L + lane) * V + i;
      w[k][i] = a.w && c < n ? wload<T>(a.w, a.wtype, c) : 1.f;
      b[k][i] = a.b && c < n ? wload<T>(a.b, a.wtype, c) : 0.f;
    }
  const float rn = 1.f / (float)n;
  for (int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L; row < a.rows; row += (int64_t)gridDim.x * G) {
    const T* x = (const T*)a.x + row * a.ldx;
    Vec<T, V> xv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * L + lane) * V;
      xv[k] = vload_n<T, V>(x + c, n - c < 0 ? 0 : n - c);
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) s += (float)xv[k].v[i];
    const float mean = group.sum(s) * rn;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = (k * L + lane) * V + i < n ? (float)xv[k].v[i] - mean : 0.f;
        s += d * d;
      }
    const float rstd = 1.f / sqrtf(group.sum(s) * rn + a.eps);
    T* y = (T*)a.y + row * n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * L + lane) * V;
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = (T)(((float)xv[k].v[i] - mean) * rstd * w[k][i] + b[k][i]);
      vstore_n<T, V>(y + c, o, n - c);
    }
    if (lane == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// rows wider than a workgroup's registers: three passes over the row, which the caches hold
template <class T>
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
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float w = a.w && i < m ? wload<T>(a.w, a.wtype, c + i) : 1.f;
        const float b = a.b && i < m ? wload<T>(a.b, a.wtype, c + i) : 0.f;
        v.v[i] = (T)(((float)v.v[i] - mean) * rstd * w + b);
      }
      vstore_n<T, V>(y + c, v, m);
    }
    if (threadIdx.x == 0 && a.mean) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// dx of every row; SUMS: one row of partial sums of dw and db a workgroup, scratch[(0 | 1)][workgroup][n]
template <class T, int L, int K, bool SUMS>
__global__ __launch_bounds__(threads_of<L>()) void layer_norm_bwd_kernel(sb_layer_norm_bwd_args a) {
  constexpr int V = vec_of<T>(), NT = threads_of<L>(), G = NT / L;
  // one column block of V values a thread at a time goes through LDS for the groups' sum
  __shared__ float lds[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float acc[SUMS && G > 1 ? NT * V : 1];
  Group<L> group{lds};
  const int lane = threadIdx.x % L;
  const int n = (int)a.n;
  float w[K][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (k * L + lane) * V + i;
      w[k][i] = a.w && c < n ? wload<T>(a.w, a.wtype, c) : 1.f;
      dw[k][i] = db[k][i] = 0.f;
    }
  const float rn = 1.f / (float)n;
  for (int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L; row < a.rows; row += (int64_t)gridDim.x * G) {
    const T* x = (const T*)a.x + row * a.ldx;
    const T* dy = (const T*)a.dy + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row];
    Vec<T, V> xv[K], gv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * L + lane) * V, m = n - c < 0 ? 0 : n - c;
      xv[k] = vload_n<T, V>(x + c, m);
      gv[k] = vload_n<T, V>(dy + c, m);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = ((float)xv[k].v[i] - mean) * rstd, g = (float)gv[k].v[i], q = g * w[k][i];
        s1 += q;
        s2 += q * xh;
        if constexpr (SUMS) {
          dw[k][i] += g * xh;
          db[k][i] += g;
        }
      }
    group.sum2(s1, s2);
    s1 *= rn;
    s2 *= rn;
    T* dx = (T*)a.dx + row * n;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * L + lane) * V;
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = ((float)xv[k].v[i] - mean) * rstd;
        o.v[i] = (T)(rstd * ((float)gv[k].v[i] * w[k][i] - s1 - xh * s2));
      }
      vstore_n<T, V>(dx + c, o, n - c);
    }
  }
  if constexpr (SUMS) {
    float* out[2] = {a.scratch + (int64_t)blockIdx.x * n, a.scratch + ((int64_t)gridDim.x + blockIdx.x) * n};
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * L + lane) * V;
        if constexpr (G == 1) {
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (c + i < n) out[which][c + i] = which ? db[k][i] : dw[k][i];
        } else {
          __syncthreads();
#pragma unroll
          for (int i = 0; i < V; ++i) acc[threadIdx.x * V + i] = which ? db[k][i] : dw[k][i];
          __syncthreads();
          for (int j = threadIdx.x; j < L * V; j += NT) {
            float s = 0.f;
            for (int g = 0; g < G; ++g) s += acc[g * L * V + j];
            if (k * L * V + j < n) out[which][k * L * V + j] = s;
          }
        }
      }
  }
}

// rows wider than a workgroup's registers: dx only, two passes over the row
template <class T>
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
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = (float)gv.v[i] * (a.w && i < m ? wload<T>(a.w, a.wtype, c + i) : 1.f);
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
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float q = (float)gv.v[i] * (a.w && i < m ? wload<T>(a.w, a.wtype, c + i) : 1.f);
        o.v[i] = (T)(rstd * (q - s1 - ((float)xv.v[i] - mean) * rstd * s2));
      }
      vstore_n<T, V>(dx + c, o, m);
    }
  }
}

// ... and the column sums of it: a thread owns a column, a workgroup a range of rows
template <class T>
__global__ __launch_bounds__(256) void layer_norm_cols_kernel(sb_layer_norm_bwd_args a, int parts) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.n) return;
  const int64_t per = (a.rows + parts - 1) / parts, r0 = blockIdx.y * per, r1 = min(a.rows, r0 + per);
  float dw = 0.f, db = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = (float)((const T*)a.dy)[r * a.lddy + c];
    dw += g * (((float)((const T*)a.x)[r * a.ldx + c] - a.mean[r]) * a.rstd[r]);
    db += g;
  }
  a.scratch[(int64_t)blockIdx.y * a.n + c] = dw;
  a.scratch[((int64_t)parts + blockIdx.y) * a.n + c] = db;
}

// dw, db from the workgroups' rows: 1024 threads are 32 columns x 32 ranges of rows
template <class T>
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float* scratch, int parts, int64_t n, int wtype, void* dw, void* db) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + col;
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const float* in = scratch + (int64_t)blockIdx.y * parts * n;
  float s = 0.f;
  if (c < n)
    for (int p = part; p < parts; p += 32) s += in[(int64_t)p * n + c];
  lds[part][col] = s;
  __syncthreads();
  if (part == 0 && c < n) {
    s = 0.f;
#pragma unroll
    for (int p = 0; p < 32; ++p) s += lds[p][col];
    if (wtype == SB_F32)
      ((float*)out)[c] = s;
    else
      ((T*)out)[c] = (T)s;
  }
}

// the group that holds a row of n elements: L lanes with K vectors each; L = 0: none does
struct Shape { int L, K; };
Shape shape_of(int64_t n, int vec, int wave_k) {
  const int64_t vecs = (n + vec - 1) / vec;
  int L = 1;
  while (L < 64 && L < vecs) L *= 2;
  int K = 1;
  const auto fit = [&](int most) {
    K = 1;
    while (K < most && (int64_t)L * K < vecs) K *= 2;
    return (int64_t)L * K >= vecs;
  };
  if (fit(wave_k)) return {L, K};
  L = 256;
  if (fit(kMaxK)) return {L, K};
  L = 1024;
  if (fit(kMaxK)) return {L, K};
  return {0, 0};
}

constexpr int kFwdWaveK = 4, kBwdWaveK = 4;

template <class T, class F> int with_shape(Shape s, F&& f) {
#define SB_CASE(l, k) \
  if (s.L == l && s.K == k) return f(std::integral_constant<int, l>(), std::integral_constant<int, k>());
  SB_CASE(1, 1) SB_CASE(2, 1) SB_CASE(4, 1) SB_CASE(8, 1) SB_CASE(16, 1) SB_CASE(32, 1) SB_CASE(64, 1) SB_CASE(64, 2) SB_CASE(64, 4)
  SB_CASE(256, 2) SB_CASE(256, 4) SB_CASE(256, 8) SB_CASE(1024, 4) SB_CASE(1024, 8)
#undef SB_CASE
  return -1009;
}

// workgroups of the backward pass = rows of partial sums
int64_t bwd_grid(int64_t rows, int64_t n, int xtype) {
  const Shape s = shape_of(n, xtype == SB_F32 ? 4 : 8, kBwdWaveK);
  if (!s.L) return std::min<int64_t>(rows, 64);
  const int64_t per = s.L >= 256 ? 1 : 256 / s.L;
  return std::min<int64_t>((rows + per - 1) / per, s.L >= 256 ? 512 : 1024);
}

}  // namespace

extern "C" int sb_layer_norm_fwd(const sb_layer_norm_args* ap, void* stream) {
  if (!ap) return -1001;
  const sb_layer_norm_args a = *ap;
  if (a.rows < 0 || a.n <= 0 || a.n > (1LL << 30) || a.ldx < 0 || (a.wtype != a.xtype && a.wtype != SB_F32)) return -1002;
  if (a.rows == 0) return 0;
  if (!a.x || !a.y || !a.mean != !a.rstd) return -1003;
  const Shape s = shape_of(a.n, a.xtype == SB_F32 ? 4 : 8, kFwdWaveK);
  return sb_with_type(a.xtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!s.L) {
      hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<T>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(1024), 0, (hipStream_t)stream, a);
    } else {
      const int rc = with_shape<T>(s, [&](auto L, auto K) -> int {
        constexpr int per = threads_of<L.value>() / L.value;
        const int64_t grid = std::min<int64_t>((a.rows + per - 1) / per, 2048);
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, L.value, K.value>), dim3((unsigned)grid), dim3(threads_of<L.value>()), 0, (hipStream_t)stream, a);
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
  const sb_layer_norm_bwd_args a = *ap;
  const bool sums = a.dw || a.db;
  if (a.rows < 0 || a.n <= 0 || a.n > (1LL << 30) || a.ldx < 0 || a.lddy < 0 || (a.wtype != a.xtype && a.wtype != SB_F32)) return -1002;
  if (a.rows > 0 && (!a.x || !a.dy || !a.dx || !a.mean || !a.rstd || (sums && !a.scratch))) return -1003;
  const Shape s = shape_of(a.n, a.xtype == SB_F32 ? 4 : 8, kBwdWaveK);
  const int grid = (int)bwd_grid(a.rows, a.n, a.xtype);
  return sb_with_type(a.xtype, [&](auto* t) -> int {
    using T = std::remove_pointer_t<decltype(t)>;
    if (a.rows > 0 && !s.L) {
      hipLaunchKernelGGL((layer_norm_bwd_wide_kernel<T>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(1024), 0, (hipStream_t)stream, a);
      SB_CHECK_LAUNCH();
      if (sums) hipLaunchKernelGGL((layer_norm_cols_kernel<T>), dim3((unsigned)((a.n + 255) / 256), grid), dim3(256), 0, (hipStream_t)stream, a, grid);
    } else if (a.rows > 0) {
      const int rc = with_shape<T>(s, [&](auto L, auto K) -> int {
        if (sums)
          hipLaunchKernelGGL((layer_norm_bwd_kernel<T, L.value, K.value, true>), dim3(grid), dim3(threads_of<L.value>()), 0, (hipStream_t)stream, a);
        else
          hipLaunchKernelGGL((layer_norm_bwd_kernel<T, L.value, K.value, false>), dim3(grid), dim3(threads_of<L.value>()), 0, (hipStream_t)stream, a);
        return 0;
      });
      if (rc) return rc;
    }
    SB_CHECK_LAUNCH();
    if (sums) {      // (no rows: no partial sums either, the sums are 0)
      hipLaunchKernelGGL((layer_norm_reduce_kernel<T>), dim3((unsigned)((a.n + 31) / 32), 2), dim3(1024), 0, (hipStream_t)stream, a.scratch,
                         a.rows > 0 ? grid : 0, a.n, a.wtype, a.dw, a.db);
      SB_CHECK_LAUNCH();
    }
    return 0;
  });
}
