// AdamW over many tensors in one launch, with 32-bit or 8-bit states, and the global norm of the
// gradients that clips it.
//
//   t <- t + 1;  s = grad_scale * clip / max(clip, |grad_scale| * norm)   (grad_scale without clipping)
//   m <- b1 m + (1 - b1) s g;  v <- b2 v + (1 - b2) (s g)^2
//   w <- w - lr wd w - lr sqrt(1 - b2^t) / (1 - b1^t) * m / (sqrt(v) + eps)
//
// A launch walks over a table of pieces (OptChunk) of at most OPT_CHUNK elements, so tensors of any
// size share it; every tensor starts at a multiple of 64 in the flat state.
//
// The step counter is OPT_MAX_GRID equal words: a workgroup reads its own and writes it (and those
// of the workgroups this launch does not have) at its end, so a captured launch counts its replays
// without an atomic, a second launch, or a word that one workgroup writes while another reads it.
//
// 8-bit states.  64 neighbouring elements of a tensor share two scale bytes, one for m and one for
// r = sqrt(v); a scale byte s is the unit 2^(s-127) of the block's codes, the smallest one with which
// the block's largest value has a code (s = 255: the block holds a value that is not finite; all
// of it reads as NaN).  A code is a small float with 4 exponent bits: m has a sign and 3 mantissa
// bits, r 4 mantissa bits, and codes below the first binade are linear, so values down to 2^-17
// (m) and 2^-18 (r) of the block's largest are told from zero.  r rather than v: it halves the range
// of exponents.  Shifted to the top of a float, a code IS the float's bits (exponent field <= 15,
// denormals for the linear part), so decoding and encoding are an ldexp and a shift.
// Rounding adds 16 bits of a hash of (place, t) below the code's last bit and cuts: with b2 = 0.999
// a second moment moves by 0.1 % a step and its code's step is 6-12 %, so it would never leave its
// code if it were rounded to the nearest.  The hash makes a step a function of its inputs alone.
// An r that is not zero keeps a code that is not zero, or m / (r + eps) would leap.
#include "adamw.h"

namespace idc {

namespace {

constexpr int TPB = 256;                         // threads of a workgroup
constexpr int ROWS = OPT_CHUNK / (TPB * 4);      // groups of 4 elements a thread takes of a chunk

struct F4 {
  float a[4];
};

__device__ __forceinline__ F4 ld4(const float* p) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  return F4{{x.x, x.y, x.z, x.w}};
}
__device__ __forceinline__ void st4(float* p, const F4& x) {
  *reinterpret_cast<float4*>(p) = make_float4(x.a[0], x.a[1], x.a[2], x.a[3]);
}
template <bool GB>
__device__ __forceinline__ F4 ldg4(const void* g, int e) {
  if constexpr (GB) {
    const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const bf16_t*>(g) + e);
    return F4{{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
               __uint_as_float(x.y & 0xffff0000u)}};
  } else {
    return ld4(reinterpret_cast<const float*>(g) + e);
  }
}
template <bool GB>
__device__ __forceinline__ float ldg1(const void* g, int e) {
  if constexpr (GB) return bf2f(reinterpret_cast<const bf16_t*>(g)[e]);
  else return reinterpret_cast<const float*>(g)[e];
}

// a piece's elements [e, e + 4), zeros from n on
template <bool GB>
__device__ __forceinline__ F4 edge_g(const void* g, int e, int n, bool vec) {
  if (vec && e + 4 <= n) return ldg4<GB>(g, e);
  F4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.a[j] = e + j < n ? ldg1<GB>(g, e + j) : 0.f;
  return r;
}
__device__ __forceinline__ F4 edge_w(const float* w, int e, int n, bool vec) {
  return edge_g<false>(w, e, n, vec);
}
__device__ __forceinline__ void edge_st(float* w, int e, int n, bool vec, const F4& x) {
  if (vec && e + 4 <= n) {
    st4(w + e, x);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (e + j < n) w[e + j] = x.a[j];
}

__device__ __forceinline__ OptChunk get_chunk(const OptChunk* p, long long go) {
  OptChunk c = *p;
  c.w = gsh(c.w, go);
  c.g = gsh(reinterpret_cast<const char*>(c.g), go);
  return c;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// the workgroup's sum, in a fixed order, for every thread
__device__ __forceinline__ double block_sum64(double v) {
  __shared__ double part[TPB / 64];
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < TPB / 64; ++i) s += part[i];
  return s;
}

// --- the codes ------------------------------------------------------------------------------
// MB mantissa bits: a code shifted by 23 - MB is a float's bits; its unit is that float's 2^-(126+MB)
template <int MB>
__device__ __forceinline__ float code_value(unsigned c, int s) {
  return ldexpf(__uint_as_float(c << (23 - MB)), s - 127 + 126 + MB);
}

// scale byte for a block whose largest magnitude has these bits: codes reach (2^(MB+1) - 1) * 2^14
template <int MB>
__device__ __forceinline__ int block_scale(unsigned top) {
  constexpr unsigned last = ((2u << MB) - 1u) << (23 - MB) & 0x7fffffu;  // mantissa of the largest code
  const int s = (int)((top + (0x7fffffu - last)) >> 23) - (14 + MB);
  return top >= 0x7f800000u ? 255 : s < 1 ? 1 : s;
}

// magnitude code of a (>= 0) with 16 random bits; a <= the block's largest
template <int MB>
__device__ __forceinline__ unsigned code_of(float a, int s, unsigned r16) {
  const unsigned x = __float_as_uint(ldexpf(a, -(s - 127 + 126 + MB)));
  return (x + (r16 << (7 - MB)) + (1u << (6 - MB))) >> (23 - MB);
}

// largest of the 16 lanes that hold a block
__device__ __forceinline__ unsigned max16(unsigned v) {
#define IDC_ROR(k) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + k, 0xf, 0xf, false))
  IDC_ROR(8);
  IDC_ROR(4);
  IDC_ROR(2);
  IDC_ROR(1);
#undef IDC_ROR
  return v;
}

constexpr unsigned HASH_STEP = 0x632BE5ABu, HASH_HIGH = 0x27D4A62Fu, HASH_1 = 0x6E7A3B15u, HASH_2 = 0x35D2C1A7u;
__device__ __forceinline__ unsigned dither(unsigned x) {
  x = (x ^ (x >> 16)) * HASH_1;
  x = (x ^ (x >> 15)) * HASH_2;
  return x ^ (x >> 16);
}

// --- one group of 4 elements -------------------------------------------------------------------
struct Hyper {
  float b1, omb1, b2, omb2, alpha, eps, scale, clip;
};

// Every product and sum of the moments is rounded by itself, in the formula's order, as the step in
// torch operations does (engine/optimizers.py, CPU): the borders between codes then lie at the same
// values on both, and a state's codes do not depend on where its step ran.
__device__ __forceinline__ void moments(F4& m, F4& v, const F4& g, float b1, float b2, const Hyper& h) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = g.a[j] * h.scale * h.clip;
    m.a[j] = b1 * m.a[j] + h.omb1 * x;
    v.a[j] = b2 * v.a[j] + h.omb2 * (x * x);
  }
}
// the decay is subtracted, not multiplied as (1 - lr wd): that factor would keep few of lr wd's bits
__device__ __forceinline__ void update(F4& w, const F4& m, const F4& root, float lr_wd, const Hyper& h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) w.a[j] -= fmaf(lr_wd, w.a[j], h.alpha * (m.a[j] / (root.a[j] + h.eps)));
}

template <int BITS>
struct State;
template <>
struct State<32> {
  F4 m, v;
  __device__ __forceinline__ void load(const AdamwArgs& a, long long i) {
    m = ld4(reinterpret_cast<const float*>(a.m) + i);
    v = ld4(reinterpret_cast<const float*>(a.v) + i);
  }
  __device__ __forceinline__ void step(const AdamwArgs& a, long long i, F4& w, const F4& g, float lr_wd,
                                       const Hyper& h, unsigned) {
    moments(m, v, g, h.b1, h.b2, h);
    F4 root;
#pragma unroll
    for (int j = 0; j < 4; ++j) root.a[j] = sqrtf(v.a[j]);
    update(w, m, root, lr_wd, h);
    st4(reinterpret_cast<float*>(a.m) + i, m);
    st4(reinterpret_cast<float*>(a.v) + i, v);
  }
};
template <>
struct State<8> {
  unsigned m4, v4;
  unsigned short sc;
  __device__ __forceinline__ void load(const AdamwArgs& a, long long i) {
    m4 = *reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned char*>(a.m) + i);
    v4 = *reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned char*>(a.v) + i);
    sc = reinterpret_cast<const unsigned short*>(a.scales)[i / OPT_BLOCK];
  }
  __device__ __forceinline__ void step(const AdamwArgs& a, long long i, F4& w, const F4& g, float lr_wd,
                                       const Hyper& h, unsigned salt) {
    const int sm = sc & 255, sv = sc >> 8;
    F4 m, v, root;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned cm = (m4 >> (8 * j)) & 255u, cv = (v4 >> (8 * j)) & 255u;
      m.a[j] = __uint_as_float(__float_as_uint(code_value<3>(cm & 127u, sm)) | ((cm & 128u) << 24));
      const float r = code_value<4>(cv, sv);
      v.a[j] = r * r;
    }
    // a block that holds no finite moment reads as NaN: through its factor
    const float nan = __uint_as_float(0x7fc00000u);
    moments(m, v, g, sm == 255 ? nan : h.b1, sv == 255 ? nan : h.b2, h);
    unsigned tm = 0, tv = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      root.a[j] = sqrtf(v.a[j]);
      tm = max(tm, __float_as_uint(m.a[j]) & 0x7fffffffu);
      tv = max(tv, __float_as_uint(root.a[j]) & 0x7fffffffu);
    }
    update(w, m, root, lr_wd, h);
    const int nm = block_scale<3>(max16(tm)), nv = block_scale<4>(max16(tv));
    const unsigned place = (unsigned)i + (unsigned)(i >> 32) * HASH_HIGH + salt;
    unsigned om = 0, ov = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned r = dither(place + j);
      const unsigned c = code_of<3>(fabsf(m.a[j]), nm, r & 0xffffu) | ((__float_as_uint(m.a[j]) >> 24) & 128u);
      const unsigned d = max(code_of<4>(root.a[j], nv, r >> 16), root.a[j] > 0.f ? 1u : 0u);
      om |= c << (8 * j);
      ov |= d << (8 * j);
    }
    *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.m) + i) = nm == 255 ? 0u : om;
    *reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.v) + i) = nv == 255 ? 0u : ov;
    if ((threadIdx.x & 15) == 0)
      reinterpret_cast<unsigned short*>(a.scales)[i / OPT_BLOCK] = (unsigned short)(nm | (nv << 8));
  }
};

template <int BITS, bool GB>
__global__ __launch_bounds__(TPB) void adamw_kernel(AdamwArgs a, GroupArg ga) {
  const long long go = goff(ga);
  a.chunks = gsh(a.chunks, go);
  a.m = gsh(reinterpret_cast<char*>(a.m), go);
  a.v = gsh(reinterpret_cast<char*>(a.v), go);
  a.scales = gsh(a.scales, go);
  a.step = gsh(a.step, go);
  a.partials = gsh(a.partials, go);
  a.norm = gsh(a.norm, go);
  a.skip = gsh(a.skip, go);
  if (a.skip && *a.skip) {  // moments, weights and the step counter stay as they are
    if (a.hostflag && (*a.skip & ~1) && blockIdx.x == 0 && threadIdx.x == 0)  // as rmsprop_kernel
      __hip_atomic_store(a.hostflag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    return;
  }
  const int t = a.step[blockIdx.x] + 1;
  Hyper h{a.b1, a.omb1, a.b2, a.omb2, 0.f, a.eps, a.grad_scale, 1.f};
  // 1 - b^t = -expm1(t log b): the product in double, so that its rounding does not grow with t
  h.alpha = a.lr * sqrtf(-expm1f((float)(t * a.log_b2))) / -expm1f((float)(t * a.log_b1));
  if (a.partials) {
    double s = 0.0;
    for (int i = threadIdx.x; i < a.npartials; i += TPB) s += a.partials[i];
    const float norm = (float)sqrt(block_sum64(s));
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    const float scaled = norm * fabsf(a.grad_scale);
    // a norm that is not finite makes every gradient NaN
    h.clip = scaled <= a.clip ? 1.f : scaled < INFINITY ? a.clip / scaled : __uint_as_float(0x7fc00000u);
  }
  const unsigned salt = (unsigned)t * HASH_STEP;
  const int e0 = threadIdx.x * 4;
  for (int c = blockIdx.x; c < a.nchunks; c += gridDim.x) {
    const OptChunk k = get_chunk(a.chunks + c, go);
    const float lr_wd = k.flags & OPT_DECAY ? a.lr_wd : 0.f;
    const bool vec = k.flags & OPT_VEC;
    State<BITS> s[ROWS];
    F4 w[ROWS], g[ROWS];
    if (vec && k.n == OPT_CHUNK) {
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        w[u] = ld4(k.w + e);
        g[u] = ldg4<GB>(k.g, e);
        s[u].load(a, k.base + e);
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        s[u].step(a, k.base + e, w[u], g[u], lr_wd, h, salt);
        st4(k.w + e, w[u]);
      }
    } else {
      // the state reaches to the next multiple of 64, so whole blocks (16 lanes) take part
      const int end = (k.n + OPT_BLOCK - 1) / OPT_BLOCK * OPT_BLOCK;
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        if (e < end) {
          w[u] = edge_w(k.w, e, k.n, vec);
          g[u] = edge_g<GB>(k.g, e, k.n, vec);
          s[u].load(a, k.base + e);
        }
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        if (e < end) {
          s[u].step(a, k.base + e, w[u], g[u], lr_wd, h, salt);
          edge_st(k.w, e, k.n, vec, w[u]);
        }
      }
    }
  }
  __syncthreads();  // every wave has read the counter
  for (int i = blockIdx.x + threadIdx.x * gridDim.x; i < OPT_MAX_GRID; i += TPB * gridDim.x) a.step[i] = t;
}

// Squares and sums in double: gradients below 1e-19 or above 1e19 have no fp32 squares, and the
// double units keep up with memory.  Each workgroup sums its pieces in a fixed order.
template <bool GB>
__device__ __forceinline__ double chunk_squares(const OptChunk& k, int e0) {
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  const bool vec = k.flags & OPT_VEC;
  F4 g[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int e = e0 + u * TPB * 4;
    if (vec && k.n == OPT_CHUNK) g[u] = ldg4<GB>(k.g, e);
    else g[u] = edge_g<GB>(k.g, e, k.n, vec);
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = fma((double)g[u].a[j], (double)g[u].a[j], s[j]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <bool GB, bool LAST>
__global__ __launch_bounds__(TPB) void grad_norm_kernel(const OptChunk* chunks, int nchunks, double* partials,
                                                        float* out, GroupArg ga) {
  const long long go = goff(ga);
  chunks = gsh(chunks, go);
  partials = gsh(partials, go);
  out = gsh(out, go);
  double s = 0.0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x)
    s += chunk_squares<GB>(get_chunk(chunks + c, go), threadIdx.x * 4);
  s = block_sum64(s);
  if (threadIdx.x == 0) {
    if (LAST) *out = (float)sqrt(s);
    else partials[blockIdx.x] = s;
  }
}

__global__ __launch_bounds__(TPB) void norm_of_partials_kernel(const double* partials, int n, float* out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += TPB) s += partials[i];
  s = block_sum64(s);
  if (threadIdx.x == 0) *out = (float)sqrt(s);
}

template <bool OB>
__global__ __launch_bounds__(TPB) void adamw_decode_kernel(const unsigned char* m, const unsigned char* v,
                                                           const unsigned char* scales, long long n4, void* om,
                                                           void* ov) {
  for (long long i = blockIdx.x * (long long)TPB + threadIdx.x; i < n4; i += (long long)gridDim.x * TPB) {
    const unsigned m4 = reinterpret_cast<const unsigned*>(m)[i], v4 = reinterpret_cast<const unsigned*>(v)[i];
    const unsigned sc = reinterpret_cast<const unsigned short*>(scales)[i / (OPT_BLOCK / 4)];
    const int sm = sc & 255, sv = sc >> 8;
    const float nan = __uint_as_float(0x7fc00000u);
    F4 x, y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned cm = (m4 >> (8 * j)) & 255u, cv = (v4 >> (8 * j)) & 255u;
      const float f = code_value<3>(cm & 127u, sm);
      x.a[j] = sm == 255 ? nan : cm & 128u ? -f : f;
      y.a[j] = sv == 255 ? nan : code_value<4>(cv, sv);
    }
    if (OB) {  // exact: at most 5 significant bits
      reinterpret_cast<uint2*>(om)[i] = make_uint2(pack2bf(x.a[0], x.a[1]), pack2bf(x.a[2], x.a[3]));
      reinterpret_cast<uint2*>(ov)[i] = make_uint2(pack2bf(y.a[0], y.a[1]), pack2bf(y.a[2], y.a[3]));
    } else {
      st4(reinterpret_cast<float*>(om) + 4 * i, x);
      st4(reinterpret_cast<float*>(ov) + 4 * i, y);
    }
  }
}

}  // namespace

hipError_t adamw(const AdamwArgs& a, int bits, int g_bf16, hipStream_t st) {
  if ((bits != 8 && bits != 32) || !a.step || a.nchunks < 0 || (a.nchunks && !(a.chunks && a.m && a.v)) ||
      (bits == 8 && a.nchunks && !a.scales) ||
      (a.partials && (!a.norm || a.npartials < 1 || a.npartials > OPT_MAX_GRID)))
    return hipErrorInvalidValue;
  const dim3 grid = ggrid(opt_grid(a.nchunks));
  if (bits == 8) {
    if (g_bf16) hipLaunchKernelGGL((adamw_kernel<8, true>), grid, dim3(TPB), 0, st, a, garg());
    else hipLaunchKernelGGL((adamw_kernel<8, false>), grid, dim3(TPB), 0, st, a, garg());
  } else {
    if (g_bf16) hipLaunchKernelGGL((adamw_kernel<32, true>), grid, dim3(TPB), 0, st, a, garg());
    else hipLaunchKernelGGL((adamw_kernel<32, false>), grid, dim3(TPB), 0, st, a, garg());
  }
  return hipGetLastError();
}

hipError_t grad_norm_partials(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, hipStream_t st) {
  if (nchunks < 0 || (nchunks && !chunks) || !partials) return hipErrorInvalidValue;
  const dim3 grid = ggrid(opt_grid(nchunks));
  if (g_bf16) hipLaunchKernelGGL((grad_norm_kernel<true, false>), grid, dim3(TPB), 0, st, chunks, nchunks, partials,
                                 (float*)nullptr, garg());
  else hipLaunchKernelGGL((grad_norm_kernel<false, false>), grid, dim3(TPB), 0, st, chunks, nchunks, partials,
                          (float*)nullptr, garg());
  return hipGetLastError();
}

hipError_t grad_norm(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, float* out, hipStream_t st) {
  if (nchunks < 0 || (nchunks && !chunks) || !partials || !out) return hipErrorInvalidValue;
  if (nchunks <= OPT_NORM_ONE) {
    if (g_bf16) hipLaunchKernelGGL((grad_norm_kernel<true, true>), dim3(1), dim3(TPB), 0, st, chunks, nchunks,
                                   partials, out, GroupArg{0, 1, 0});
    else hipLaunchKernelGGL((grad_norm_kernel<false, true>), dim3(1), dim3(TPB), 0, st, chunks, nchunks, partials,
                            out, GroupArg{0, 1, 0});
    return hipGetLastError();
  }
  const int grid = opt_grid(nchunks);
  if (g_bf16) hipLaunchKernelGGL((grad_norm_kernel<true, false>), dim3(grid), dim3(TPB), 0, st, chunks, nchunks,
                                 partials, (float*)nullptr, GroupArg{0, 1, 0});
  else hipLaunchKernelGGL((grad_norm_kernel<false, false>), dim3(grid), dim3(TPB), 0, st, chunks, nchunks, partials,
                          (float*)nullptr, GroupArg{0, 1, 0});
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(norm_of_partials_kernel, dim3(1), dim3(TPB), 0, st, partials, grid, out);
  return hipGetLastError();
}

hipError_t adamw_decode(const unsigned char* m, const unsigned char* v, const unsigned char* scales, long long n,
                        void* om, void* ov, int out_bf16, hipStream_t st) {
  if (n < 0 || n % OPT_BLOCK) return hipErrorInvalidValue;
  if (n == 0) return hipSuccess;
  if (!m || !v || !scales || !om || !ov) return hipErrorInvalidValue;
  const long long n4 = n / 4, blocks = (n4 + TPB - 1) / TPB;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  if (out_bf16) hipLaunchKernelGGL(adamw_decode_kernel<true>, grid, dim3(TPB), 0, st, m, v, scales, n4, om, ov);
  else hipLaunchKernelGGL(adamw_decode_kernel<false>, grid, dim3(TPB), 0, st, m, v, scales, n4, om, ov);
  return hipGetLastError();
}

}  // namespace idc
