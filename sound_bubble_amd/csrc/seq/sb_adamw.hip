// AdamW over many tensors in one launch, states in fp32 or in 8 bits, and the sum of squares for the gradient's clipping.
//
// A launch's tensors come as a table in the kernel's arguments; a workgroup takes chunks of kChunk elements, a wave blocks of 256
// (4 elements a lane), the unit that shares a scale where the states are in 8 bits.  Every operation is rounded by itself (the file is
// compiled without contraction), so that the value a code is made from is the formula's own.
#include "sb_seq_common.h"

namespace {

constexpr int kBlock = SB_ADAMW_BLOCK, kChunk = 4096, kPerWave = kChunk / kBlock / 4;      // blocks of a wave in a chunk
static_assert(kBlock == 64 * 4, "a wave holds a block");

SB_DEVINL double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}
// sum over the workgroup's 4 waves, in every thread
SB_DEVINL double block_sum_f64(double v, double* lds) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}
// the largest bit pattern of |x| in the wave: NaN and infinity come out on top
SB_DEVINL unsigned wave_max_bits(unsigned v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = max(v, (unsigned)__shfl_xor((int)v, d, 64));
  return v;
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

template <class G> __global__ __launch_bounds__(256) void adamw_norm_kernel(sb_adamw_args a, double* part, int chunks) {
  __shared__ double lds[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const sb_adamw_tensor& t = a.t[tensor_of(a, c)];
    const int64_t i0 = (int64_t)(c - t.first_chunk) * kChunk;
    const G* g = (const G*)t.g;
#pragma unroll
    for (int j = 0; j < kChunk / 1024; ++j) {
      const int64_t i = i0 + j * 1024 + threadIdx.x * 4;
      const Vec<G, 4> v = vload_n<G, 4>(g + i, (int)min(max(t.n - i, (int64_t)0), (int64_t)4));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double d = (double)(float)v.v[k];
        s += d * d;
      }
    }
  }
  s = block_sum_f64(s, lds);
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
  static SB_DEVINL float inverse(int byte) { return __int_as_float((254 - byte) << 23); }
  // |x| / scale as y >= 0 to a code: up where the part cut off and (u16 + 1/2) / 2^16 reach 1
  static SB_DEVINL unsigned code(float y, unsigned u16) {
    constexpr int CUT = 23 - M;
    const unsigned add = (u16 << (CUT - 16)) + (1u << (CUT - 17));
    constexpr float lowest = 1.f / (float)(1 << (BIAS - 1));
    if (y >= lowest) return (((unsigned)__float_as_int(y) + add) >> CUT) - ((127 - BIAS) << M);
    return ((unsigned)(y * __int_as_float((127 + BIAS - 1 + M + CUT) << 23)) + add) >> CUT;
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
    const float norm = sqrtf((float)block_sum_f64(s, lds)) * a.gscale;
    const float coef = a.clip / (norm + 1e-6f);
    r.gscale *= coef > 1.f ? 1.f : coef;      // (a NaN norm stays one)
  }
  return r;
}

template <class P, class G, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(sb_adamw_args a, int chunks) {
  __shared__ double lds[4];
  if (a.guard && __hip_atomic_load(a.guard, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0) {
    if (a.last && a.skipped && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(a.skipped, 1);
    return;
  }
  const Rates r = rates_of(a, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr bool kMaster = !std::is_same_v<P, float>;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const sb_adamw_tensor& t = a.t[tensor_of(a, c)];
    const int64_t i0 = (int64_t)(c - t.first_chunk) * kChunk + wave * (kPerWave * kBlock);
    const int64_t s0 = (int64_t)t.first_block * kBlock + i0;
    P* pp = (P*)t.p;
    const G* gp = (const G*)t.g;
#pragma unroll
    for (int j = 0; j < kPerWave; ++j) {
      const int64_t i = i0 + j * kBlock + lane * 4, s = s0 + j * kBlock + lane * 4;
      if (i0 + j * kBlock >= t.n) break;      // (the whole wave)
      const int n = (int)min(max(t.n - i, (int64_t)0), (int64_t)4);
      const Vec<G, 4> gv = vload_n<G, 4>(gp + i, n);
      Vec<float, 4> p, m, v;
      if constexpr (kMaster) {
        p = vload_n<float, 4>(a.master + s, n);
      } else {
        p = vload_n<float, 4>(pp + i, n);
      }
      if constexpr (BITS == 32) {
        m = vload_n<float, 4>((const float*)a.m + s, n);
        v = vload_n<float, 4>((const float*)a.v + s, n);
      } else {
        const int mc = *(const int*)((const uint8_t*)a.m + s), vc = *(const int*)((const uint8_t*)a.v + s);
        const float ms = E4M3::scale(((const uint8_t*)a.m_scale)[s / kBlock]), vs = E5M2::scale(((const uint8_t*)a.v_scale)[s / kBlock]);
        m.v[0] = __builtin_amdgcn_cvt_f32_fp8(mc, 0) * ms;
        m.v[1] = __builtin_amdgcn_cvt_f32_fp8(mc, 1) * ms;
        m.v[2] = __builtin_amdgcn_cvt_f32_fp8(mc, 2) * ms;
        m.v[3] = __builtin_amdgcn_cvt_f32_fp8(mc, 3) * ms;
        v.v[0] = __builtin_amdgcn_cvt_f32_bf8(vc, 0) * vs;
        v.v[1] = __builtin_amdgcn_cvt_f32_bf8(vc, 1) * vs;
        v.v[2] = __builtin_amdgcn_cvt_f32_bf8(vc, 2) * vs;
        v.v[3] = __builtin_amdgcn_cvt_f32_bf8(vc, 3) * vs;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float g = (float)gv.v[k] * r.gscale;
        m.v[k] = m.v[k] * r.b1 + g * r.c1;
        v.v[k] = v.v[k] * r.b2 + (g * g) * r.c2;
        const float u = m.v[k] / (sqrtf(v.v[k]) * r.root2 + r.eps);
        p.v[k] = p.v[k] * r.decay - r.rate * u;
        if (k >= n) m.v[k] = v.v[k] = 0.f;
      }
      if constexpr (kMaster) {
        vstore_n<float, 4>(a.master + s, p, n);
        Vec<P, 4> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.v[k] = (P)p.v[k];
        vstore_n<P, 4>(pp + i, o, n);
      } else {
        vstore_n<float, 4>(pp + i, p, n);
      }
      if constexpr (BITS == 32) {
        vstore_n<float, 4>((float*)a.m + s, m, n);
        vstore_n<float, 4>((float*)a.v + s, v, n);
      } else {
        unsigned mb = 0, vb = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          mb = max(mb, (unsigned)__float_as_int(m.v[k]) & 0x7FFFFFFFu);
          vb = max(vb, (unsigned)__float_as_int(v.v[k]) & 0x7FFFFFFFu);
        }
        const int ms = E4M3::scale_byte(wave_max_bits(mb)), vs = E5M2::scale_byte(wave_max_bits(vb));
        unsigned mc = 0, vc = 0;
        const float mi = E4M3::inverse(ms), vi = E5M2::inverse(vs);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned u = dither(s + k, r.key);
          unsigned q = E4M3::code(__builtin_fabsf(m.v[k]) * mi, u & 0xFFFFu) | ((unsigned)__float_as_int(m.v[k]) >> 31 << 7);
          mc |= (ms == 255 ? 0u : q) << (8 * k);
          q = E5M2::code(v.v[k] * vi, u >> 16);
          if (q == 0 && v.v[k] > 0.f) q = 1;
          vc |= (vs == 255 ? 0u : q) << (8 * k);
        }
        *(unsigned*)((uint8_t*)a.m + s) = mc;
        *(unsigned*)((uint8_t*)a.v + s) = vc;
        if (lane == 0) {
          ((uint8_t*)a.m_scale)[s / kBlock] = (uint8_t)ms;
          ((uint8_t*)a.v_scale)[s / kBlock] = (uint8_t)vs;
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

constexpr int kGrid = 2048;

}  // namespace

extern "C" int sb_adamw_chunk(void) { return kChunk; }

extern "C" int sb_adamw_norm(const sb_adamw_args* a, double* norm_part, int slot0, int slots, void* stream) {
  if (!a || !norm_part || slot0 < 0 || slots <= 0 || slot0 + slots > SB_ADAMW_NORM_SLOTS) return -1001;
  const int64_t chunks = chunks_of(*a, false);
  if (chunks < 0) return (int)chunks;
  return sb_with_type(a->gtype, [&](auto* t) -> int {
    using G = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((adamw_norm_kernel<G>), dim3(slots), dim3(256), 0, (hipStream_t)stream, *a, norm_part + slot0, (int)chunks);
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
  if ((!a->step_dev && a->step <= 0) || a->clip < 0.f || (a->clip > 0.f && (!a->norm_part || a->norm_slots <= 0 || a->norm_slots > SB_ADAMW_NORM_SLOTS)))
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
