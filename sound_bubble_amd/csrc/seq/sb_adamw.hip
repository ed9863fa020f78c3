// AdamW over many tensors in one launch, states in fp32 or in 8 bits, and the sum of squares for the gradient's clipping.
//
// A launch's tensors come as a table in the kernel's arguments; a workgroup takes chunks of kChunk elements, a wave blocks of 256
// (4 elements a lane), the unit that shares a scale where the states are in 8 bits.  Every operation is rounded by itself (the file is
// compiled without contraction), so that the value a code is made from is the formula's own; the update itself, which no code is made
// from, takes the hardware's square root and reciprocal (1 ulp each).
#include "sb_seq_common.h"

namespace {

constexpr int kBlock = SB_ADAMW_BLOCK, kChunk = 8192, kPerWave = kChunk / kBlock / 4;      // blocks of a wave in a chunk
constexpr int kTogether = 4;      // blocks whose loads are under way together
constexpr int kNormThreads = 512;
static_assert(kBlock == 64 * 4, "a wave holds a block");

SB_DEVINL double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}
// sum over the workgroup's N waves, in every thread
template <int N> SB_DEVINL double block_sum_f64(double v, double* lds) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < N; ++w) s += lds[w];
  return s;
}
// the largest bit pattern of |x| in the wave, uniform: NaN and infinity come out on top
template <int CTRL> SB_DEVINL unsigned dpp_max(unsigned v) { return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false)); }
SB_DEVINL unsigned wave_max_bits(unsigned v) {
  v = dpp_max<0xB1>(v);      // quad_perm [1,0,3,2]
  v = dpp_max<0x4E>(v);      // quad_perm [2,3,0,1]
  v = dpp_max<0x141>(v);     // row_half_mirror
  v = dpp_max<0x140>(v);     // row_mirror
  const unsigned a = max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16));
  return max(a, max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}

// the tensor that chunk `c` of the launch belongs to
SB_DEVINL int tensor_of(const sb_adamw_args& a, int c) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.t[mid].first_chunk <= c) lo = mid; else hi = mid;
  }
  return lo;
}

template <class G> __global__ __launch_bounds__(kNormThreads) void adamw_norm_kernel(sb_adamw_args a, double* part, int chunks) {
  __shared__ double lds[kNormThreads / 64];
  constexpr int V = vec_of<G>(), N = kChunk / kNormThreads / V;
  double s = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const sb_adamw_tensor& t = a.t[tensor_of(a, c)];
    const int64_t i0 = (int64_t)(c - t.first_chunk) * kChunk;
    const G* g = (const G*)t.g + i0;
    const int n = (int)min(t.n - i0, (int64_t)kChunk);
    Vec<G, V> v[N];
    if (n == kChunk) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = vload<G, V>(g + (j * kNormThreads + threadIdx.x) * V);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = (j * kNormThreads + threadIdx.x) * V;
        v[j] = vload_n<G, V>(g + i, max(n - i, 0));
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double d = (double)(float)v[j].v[k];
        s += d * d;
      }
  }
  s = block_sum_f64<kNormThreads / 64>(s, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// 32 bits for an element of the buffers: Weyl sequence over the index, two multiply-xorshift rounds
SB_DEVINL unsigned dither(int64_t i, unsigned key) {
  unsigned x = (unsigned)i + (unsigned)(i >> 32) * 0x3C6EF372u + key;
  x = (x ^ (x >> 16)) * 0x5BE0CD19u;
  x = (x ^ (x >> 15)) * 0x1F83D9ABu;
  return x ^ (x >> 16);
}

// 8-bit floats with a shared scale 2^(byte - 127): M mantissa bits, exponent bias, exponent of the largest code (its mantissa is 1.75)
template <int M, int BIAS, int TOP> struct Float8 {
  // the scale's byte for a block whose largest |x| has these bits
  static SB_DEVINL int scale_byte(unsigned big) {
    if (big >= 0x7F800000u) return 255;
    const int e = (int)(big >> 23) - 127 + ((big & 0x7FFFFFu) > 0x600000u ? 1 : 0) - TOP;
    return max(e, -127) + 127;
  }
  static SB_DEVINL float scale(int byte) {
    return byte == 255 ? __builtin_nanf("") : __int_as_float(byte ? byte << 23 : 1 << 22);
  }
  // 2^(127 - byte): exact, as the format says (a power function need not be)
  static SB_DEVINL float inverse(int byte) { return __int_as_float((254 - byte) << 23); }
  // |x| / scale as y >= 0 to a code: up where the part cut off and (u16 + 1/2) / 2^16 reach 1
  static SB_DEVINL unsigned code(float y, unsigned u16) {
    constexpr int CUT = 23 - M;
    const unsigned add = (u16 << (CUT - 16)) + (1u << (CUT - 17));
    constexpr float lowest = 1.f / (float)(1 << (BIAS - 1));
    const unsigned normal = (((unsigned)__float_as_int(y) + add) >> CUT) - ((127 - BIAS) << M);
    const unsigned small = ((unsigned)(y * __int_as_float((127 + BIAS - 1 + M + CUT) << 23)) + add) >> CUT;
    return y >= lowest ? normal : small;
  }
};
using E4M3 = Float8<3, 7, 8>;
using E5M2 = Float8<2, 15, 15>;

struct Rates { float b1, c1, b2, c2, decay, rate, root2, eps, gscale; unsigned key; };

SB_DEVINL Rates rates_of(const sb_adamw_args& a, double* lds) {
  Rates r;
  const int step = a.step_dev ? *a.step_dev : a.step;
  const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
  double p1 = 1.0, p2 = 1.0, q1 = a.beta1, q2 = a.beta2;
  for (unsigned n = (unsigned)step; n; n >>= 1) {      // beta^step
    if (n & 1) {
      p1 *= q1;
      p2 *= q2;
    }
    q1 *= q1;
    q2 *= q2;
  }
  r.b1 = (float)a.beta1;
  r.c1 = (float)(1.0 - a.beta1);
  r.b2 = (float)a.beta2;
  r.c2 = (float)(1.0 - a.beta2);
  r.decay = (float)(1.0 - lr * a.weight_decay);
  r.rate = (float)(lr / (1.0 - p1));
  r.root2 = (float)(1.0 / sqrt(1.0 - p2));
  r.eps = (float)a.eps;
  r.gscale = a.gscale;
  r.key = a.seed * 0x9E3779B9u + (unsigned)step * 0x6A09E667u;
  if (a.clip > 0.f) {
    double s = 0.0;
    for (int i = threadIdx.x; i < a.norm_slots; i += 256) s += a.norm_part[i];
    s = block_sum_f64<4>(s, lds);
    // (a sum beyond float32 has a root well within it: finite gradients of 1e20 are clipped, not dropped)
    const float coef = s > 3.402823466e38 ? (float)(a.clip / (sqrt(s) * a.gscale + 1e-6)) : a.clip / (sqrtf((float)s) * a.gscale + 1e-6f);
    r.gscale *= coef > 1.f ? 1.f : coef;      // (a NaN norm stays one)
  }
  return r;
}

// Read once and written once: streams past the caches.  96 M bf16 parameters with fp32 states, us: plain 640, stores so 626, loads too 546
template <class E> SB_DEVINL Vec<E, 4> stream_load(const E* p) {
  typedef E x4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));
  const x4 v = __builtin_nontemporal_load((const x4*)p);
  return {v[0], v[1], v[2], v[3]};
}
template <class E> SB_DEVINL void stream_store(E* p, const Vec<E, 4>& o) {
  typedef E x4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));
  const x4 v = {o.v[0], o.v[1], o.v[2], o.v[3]};
  __builtin_nontemporal_store(v, (x4*)p);
}

// sqrt(v); the hardware's counts v below 2^-126 as 0, which under an eps of 0 makes an infinite update of one of about lr: those are taken
// 2^64 times as large
SB_DEVINL float root(float v) {
  const bool low = v < 1.17549435e-38f;
  const float s = __builtin_amdgcn_sqrtf(low ? v * 18446744073709551616.f : v);
  return low ? s * 2.3283064365386963e-10f : s;
}

// what a lane holds of a block: 4 elements
template <class P, class G, int BITS> struct Part {
  static constexpr bool kMaster = !std::is_same_v<P, float>;
  Vec<G, 4> g;
  Vec<float, 4> p, m, v;
  int mc, vc, ms, vs;

  // n: elements that exist, 4 where FULL
  template <bool FULL> SB_DEVINL void load(const sb_adamw_args& a, const P* pp, const G* gp, int64_t i, int64_t s, int n) {
    g = FULL ? stream_load(gp + i) : vload_n<G, 4>(gp + i, n);
    const float* from = kMaster ? a.master + s : (const float*)pp + i;
    p = FULL ? stream_load(from) : vload_n<float, 4>(from, n);
    if constexpr (BITS == 32) {
      m = FULL ? stream_load((const float*)a.m + s) : vload_n<float, 4>((const float*)a.m + s, n);
      v = FULL ? stream_load((const float*)a.v + s) : vload_n<float, 4>((const float*)a.v + s, n);
    } else {      // (the buffers have whole blocks)
      mc = __builtin_nontemporal_load((const int*)((const uint8_t*)a.m + s));
      vc = __builtin_nontemporal_load((const int*)((const uint8_t*)a.v + s));
      ms = ((const uint8_t*)a.m_scale)[s / kBlock];
      vs = ((const uint8_t*)a.v_scale)[s / kBlock];
    }
  }
  SB_DEVINL void step(const Rates& r, int n) {
    if constexpr (BITS == 8) {
      const float mf = E4M3::scale(ms), vf = E5M2::scale(vs);
      m.v[0] = __builtin_amdgcn_cvt_f32_fp8(mc, 0) * mf;
      m.v[1] = __builtin_amdgcn_cvt_f32_fp8(mc, 1) * mf;
      m.v[2] = __builtin_amdgcn_cvt_f32_fp8(mc, 2) * mf;
      m.v[3] = __builtin_amdgcn_cvt_f32_fp8(mc, 3) * mf;
      v.v[0] = __builtin_amdgcn_cvt_f32_bf8(vc, 0) * vf;
      v.v[1] = __builtin_amdgcn_cvt_f32_bf8(vc, 1) * vf;
      v.v[2] = __builtin_amdgcn_cvt_f32_bf8(vc, 2) * vf;
      v.v[3] = __builtin_amdgcn_cvt_f32_bf8(vc, 3) * vf;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = (float)g.v[k] * r.gscale;
      m.v[k] = m.v[k] * r.b1 + f * r.c1;
      v.v[k] = v.v[k] * r.b2 + (f * f) * r.c2;
      p.v[k] = p.v[k] * r.decay - r.rate * (m.v[k] * __builtin_amdgcn_rcpf(root(v.v[k]) * r.root2 + r.eps));
      if (k >= n) m.v[k] = v.v[k] = 0.f;
    }
  }
  template <bool FULL> SB_DEVINL void store(const sb_adamw_args& a, const Rates& r, P* pp, int64_t i, int64_t s, int n) {
    if constexpr (kMaster) {
      Vec<P, 4> o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o.v[k] = (P)p.v[k];
      if constexpr (FULL) stream_store(pp + i, o); else vstore_n<P, 4>(pp + i, o, n);
    }
    float* to = kMaster ? a.master + s : (float*)pp + i;
    if constexpr (FULL) stream_store(to, p); else vstore_n<float, 4>(to, p, n);
    if constexpr (BITS == 32) {
      if constexpr (FULL) stream_store((float*)a.m + s, m); else vstore_n<float, 4>((float*)a.m + s, m, n);
      if constexpr (FULL) stream_store((float*)a.v + s, v); else vstore_n<float, 4>((float*)a.v + s, v, n);
    } else {
      unsigned mb = 0, vb = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mb = max(mb, (unsigned)__float_as_int(m.v[k]) & 0x7FFFFFFFu);
        vb = max(vb, (unsigned)__float_as_int(v.v[k]) & 0x7FFFFFFFu);
      }
      const int mscale = E4M3::scale_byte(wave_max_bits(mb)), vscale = E5M2::scale_byte(wave_max_bits(vb));
      unsigned mq = 0, vq = 0;
      const float mi = E4M3::inverse(mscale), vi = E5M2::inverse(vscale);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned u = dither(s + k, r.key);
        unsigned q = E4M3::code(__builtin_fabsf(m.v[k]) * mi, u & 0xFFFFu) | ((unsigned)__float_as_int(m.v[k]) >> 31 << 7);
        mq |= (mscale == 255 ? 0u : q) << (8 * k);
        q = E5M2::code(v.v[k] * vi, u >> 16);
        if (q == 0 && v.v[k] > 0.f) q = 1;
        vq |= (vscale == 255 ? 0u : q) << (8 * k);
      }
      *(unsigned*)((uint8_t*)a.m + s) = mq;
      *(unsigned*)((uint8_t*)a.v + s) = vq;
      if ((threadIdx.x & 63) == 0) {
        ((uint8_t*)a.m_scale)[s / kBlock] = (uint8_t)mscale;
        ((uint8_t*)a.v_scale)[s / kBlock] = (uint8_t)vscale;
      }
    }
  }
};

template <class P, class G, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(sb_adamw_args a, int chunks) {
  __shared__ double lds[4];
  if (a.guard && __hip_atomic_load(a.guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0) {
    if (a.last && a.skipped && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(a.skipped, 1);
    return;
  }
  const Rates r = rates_of(a, lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const sb_adamw_tensor& t = a.t[tensor_of(a, c)];
    const int64_t i0 = (int64_t)(c - t.first_chunk) * kChunk + wave * (kPerWave * kBlock);
    const int64_t s0 = (int64_t)t.first_block * kBlock + i0;
    P* pp = (P*)t.p;
    const G* gp = (const G*)t.g;
    for (int j = 0; j < kPerWave && i0 + j * kBlock < t.n; j += kTogether) {
      const int64_t i = i0 + j * kBlock + lane * 4, s = s0 + j * kBlock + lane * 4;
      Part<P, G, BITS> part[kTogether];
      if (i0 + (j + kTogether) * kBlock <= t.n) {
#pragma unroll
        for (int b = 0; b < kTogether; ++b) part[b].template load<true>(a, pp, gp, i + b * kBlock, s + b * kBlock, 4);
#pragma unroll
        for (int b = 0; b < kTogether; ++b) part[b].step(r, 4);
#pragma unroll
        for (int b = 0; b < kTogether; ++b) part[b].template store<true>(a, r, pp, i + b * kBlock, s + b * kBlock, 4);
      } else {
        for (int b = 0; b < kTogether && i0 + (j + b) * kBlock < t.n; ++b) {      // (the whole wave)
          const int n = (int)min(max(t.n - i - b * kBlock, (int64_t)0), (int64_t)4);
          part[0].template load<false>(a, pp, gp, i + b * kBlock, s + b * kBlock, n);
          part[0].step(r, n);
          part[0].template store<false>(a, r, pp, i + b * kBlock, s + b * kBlock, n);
        }
      }
    }
  }
}

// chunks of the launch, < 0: a bad table
int64_t chunks_of(const sb_adamw_args& a, bool step) {
  if (a.count <= 0 || a.count > SB_ADAMW_MAX) return -1002;
  int64_t chunks = 0;
  for (int i = 0; i < a.count; ++i) {
    const sb_adamw_tensor& t = a.t[i];
    if (t.n <= 0 || !t.g || t.first_chunk != chunks || (step && (!t.p || t.first_block < 0))) return -1003;
    chunks += (t.n + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffffLL) return -1004;
  }
  return chunks;
}

constexpr int kGrid = 4096;

}  // namespace

extern "C" int sb_adamw_chunk(void) { return kChunk; }

extern "C" int sb_adamw_norm(const sb_adamw_args* a, double* norm_part, int slot0, int slots, void* stream) {
  if (!a || !norm_part || slot0 < 0 || slots <= 0 || slot0 + slots > SB_ADAMW_NORM_SLOTS) return -1001;
  const int64_t chunks = chunks_of(*a, false);
  if (chunks < 0) return (int)chunks;
  return sb_with_type(a->gtype, [&](auto* t) -> int {
    using G = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((adamw_norm_kernel<G>), dim3(slots), dim3(kNormThreads), 0, (hipStream_t)stream, *a, norm_part + slot0, (int)chunks);
    SB_CHECK_LAUNCH();
    return 0;
  });
}

extern "C" int sb_adamw_step(const sb_adamw_args* a, void* stream) {
  if (!a) return -1001;
  const int64_t chunks = chunks_of(*a, true);
  if (chunks < 0) return (int)chunks;
  if ((a->bits != 32 && a->bits != 8) || !a->m || !a->v || (a->bits == 8 && (!a->m_scale || !a->v_scale))) return -1005;
  if ((a->ptype != SB_F32 && !a->master) || (a->gtype != a->ptype && a->gtype != SB_F32)) return -1006;
  if ((!a->step_dev && a->step <= 0) || !(a->clip >= 0.f) || (a->clip > 0.f && (!a->norm_part || a->norm_slots <= 0 || a->norm_slots > SB_ADAMW_NORM_SLOTS)))
    return -1007;
  const int grid = (int)std::min<int64_t>(chunks, kGrid);
  return sb_with_type(a->ptype, [&](auto* pt) -> int {
    using P = std::remove_pointer_t<decltype(pt)>;
    const auto go = [&](auto* gt) -> int {
      using G = std::remove_pointer_t<decltype(gt)>;
      if (a->bits == 32)
        hipLaunchKernelGGL((adamw_kernel<P, G, 32>), dim3(grid), dim3(256), 0, (hipStream_t)stream, *a, (int)chunks);
      else
        hipLaunchKernelGGL((adamw_kernel<P, G, 8>), dim3(grid), dim3(256), 0, (hipStream_t)stream, *a, (int)chunks);
      SB_CHECK_LAUNCH();
      return 0;
    };
    if (a->gtype == a->ptype) return go(pt);
    return go((float*)nullptr);
  });
}
