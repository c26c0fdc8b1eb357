// AdamW over many tensors in one launch, with 32-bit or 8-bit states, and the global norm of the
// gradients that clips it.
//
//   t <- t + 1;  s = grad_scale * clip / max(clip, |grad_scale| * norm)   (grad_scale without clipping)
//   m <- b1 m + (1 - b1) s g;  v <- b2 v + (1 - b2) (s g)^2
//   w <- w - lr wd w - lr sqrt(1 - b2^t) / (1 - b1^t) * m / (sqrt(v) + eps)
//
// A launch walks over a table of pieces (OptChunk) of at most 2048 or 4096 elements, so tensors of any
// size share it; every tensor starts at a multiple of 64 in the flat state.  Memory bounds it: 24 bytes a
// weight and the gradient's 4 or 2 (32-bit states), or 12 and the gradient's (8-bit); 120M weights with bf16
// gradients take 518 us on the device (6.0 TB/s) and 268 us (6.3 TB/s).
//
// The step counter is OPT_MAX_GRID equal words: a workgroup reads its own and writes it (and those
// of the workgroups this launch does not have) at its end, so a captured launch counts its replays
// without an atomic, a second launch, or a word that one workgroup writes while another reads it.  (The
// largest tables have a launch of one workgroup ahead that counts: adamw_begin_kernel.)
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

constexpr int TPB = 256;  // threads of a workgroup; a row is the TPB * 4 elements they take at once

struct F4 {
  float a[4];
};
typedef float vf4 __attribute__((ext_vector_type(4)));

// NT: past the caches (see `adamw`)
template <bool NT = false, typename T>
__device__ __forceinline__ T ld(const T* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool NT = false, typename T>
__device__ __forceinline__ void st(T* p, T x) {
  if constexpr (NT) __builtin_nontemporal_store(x, p);
  else *p = x;
}
template <bool NT = false>
__device__ __forceinline__ F4 ld4(const float* p) {
  const vf4 x = ld<NT>(reinterpret_cast<const vf4*>(p));
  return F4{{x.x, x.y, x.z, x.w}};
}
template <bool NT = false>
__device__ __forceinline__ void st4(float* p, const F4& x) {
  st<NT>(reinterpret_cast<vf4*>(p), vf4{x.a[0], x.a[1], x.a[2], x.a[3]});
}
template <bool GB, bool NT = false>
__device__ __forceinline__ F4 ldg4(const void* g, int e) {
  if constexpr (GB) {
    typedef unsigned vu2 __attribute__((ext_vector_type(2)));
    const vu2 x = ld<NT>(reinterpret_cast<const vu2*>(reinterpret_cast<const bf16_t*>(g) + e));
    return F4{{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
               __uint_as_float(x.y & 0xffff0000u)}};
  } else {
    return ld4<NT>(reinterpret_cast<const float*>(g) + e);
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
// A code of MB mantissa bits, its bits at a float's place (shifted by 23 - MB), times 2^(126+MB) is
// its value in units; the unit is 2^(s-127).
template <int MB>
__device__ __forceinline__ float code_value(unsigned x, int s) {
  return ldexpf(__uint_as_float(x), s - 127 + 126 + MB);
}
// byte j of a word of first moments (sign and 7 bits), and of a word of roots
template <int J>
__device__ __forceinline__ float m_value(unsigned word, int s) {
  return code_value<3>((unsigned)((int)(word << (24 - 8 * J)) >> 4) & 0x87f00000u, s);
}
template <int J>
__device__ __forceinline__ float root_value(unsigned word, int s) {
  return code_value<4>((word >> (8 * J) & 255u) << 19, s);
}

// scale byte for a block whose largest magnitude has these bits: codes reach (2^(MB+1) - 1) * 2^14
template <int MB>
__device__ __forceinline__ int block_scale(unsigned top) {
  constexpr unsigned last = (((2u << MB) - 1u) << (23 - MB)) & 0x7fffffu;  // mantissa of the largest code
  const int s = (int)((top + (0x7fffffu - last)) >> 23) - (14 + MB);
  return top >= 0x7f800000u ? 255 : s < 1 ? 1 : s;
}

// the code of |a| <= the block's largest, in the bits from 23 - MB on (what is below is left over);
// bits: 16 random ones, in the bits from 7 - MB on, and the half of the last of them
template <int MB>
__device__ __forceinline__ unsigned code_of(float a, int s, unsigned bits) {
  return __float_as_uint(ldexpf(fabsf(a), -(s - 127 + 126 + MB))) + bits;
}

__device__ __forceinline__ unsigned top_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0703u), __builtin_amdgcn_perm(b, a, 0x0c0c0703u), 0x05040100u);
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
// The decay is subtracted, not multiplied as (1 - lr wd): that factor would keep few of lr wd's bits.
// The quotient is a reciprocal (to one unit in its last place) and a product: 3 half steps of fp32 in
// the update, which a weight's own rounding hides, for a third of a division's instructions (8-bit states,
// 7M weights: 23.3 -> 21.1 us).  eps is a normal number, and so is what is inverted.
__device__ __forceinline__ void update(F4& w, const F4& m, const F4& root, float lr_wd, const Hyper& h) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w.a[j] -= fmaf(lr_wd, w.a[j], h.alpha * (m.a[j] * __builtin_amdgcn_rcpf(root.a[j] + h.eps)));
}

template <int BITS, bool NT>
struct State;
template <bool NT>
struct State<32, NT> {
  F4 m, v;
  __device__ __forceinline__ void load(const AdamwArgs& a, long long i) {
    m = ld4<NT>(reinterpret_cast<const float*>(a.m) + i);
    v = ld4<NT>(reinterpret_cast<const float*>(a.v) + i);
  }
  __device__ __forceinline__ void step(const AdamwArgs& a, long long i, F4& w, const F4& g, float lr_wd,
                                       const Hyper& h, unsigned) {
    moments(m, v, g, h.b1, h.b2, h);
    F4 root;
#pragma unroll
    for (int j = 0; j < 4; ++j) root.a[j] = sqrtf(v.a[j]);
    update(w, m, root, lr_wd, h);
    st4<NT>(reinterpret_cast<float*>(a.m) + i, m);
    st4<NT>(reinterpret_cast<float*>(a.v) + i, v);
  }
};
template <bool NT>
struct State<8, NT> {
  unsigned m4, v4;
  unsigned short sc;
  __device__ __forceinline__ void load(const AdamwArgs& a, long long i) {
    m4 = ld<NT>(reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned char*>(a.m) + i));
    v4 = ld<NT>(reinterpret_cast<const unsigned*>(reinterpret_cast<const unsigned char*>(a.v) + i));
    sc = reinterpret_cast<const unsigned short*>(a.scales)[i / OPT_BLOCK];
  }
  __device__ __forceinline__ void step(const AdamwArgs& a, long long i, F4& w, const F4& g, float lr_wd,
                                       const Hyper& h, unsigned salt) {
    const int sm = sc & 255, sv = sc >> 8;
    F4 m = {{m_value<0>(m4, sm), m_value<1>(m4, sm), m_value<2>(m4, sm), m_value<3>(m4, sm)}};
    F4 root = {{root_value<0>(v4, sv), root_value<1>(v4, sv), root_value<2>(v4, sv), root_value<3>(v4, sv)}};
    F4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v.a[j] = root.a[j] * root.a[j];
    // a block that holds a moment that is not finite reads as NaN: through its factor
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
    unsigned c[4], d[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned r = dither(place + j);
      // codes to the top byte of a word: the sign over 7 bits, or 8 bits
      c[j] = (code_of<3>(m.a[j], nm, (r << 16 | 0x8000u) >> 12) << 4 & 0x7fffffffu) | (__float_as_uint(m.a[j]) & 0x80000000u);
      d[j] = max(code_of<4>(root.a[j], nv, (r >> 13 & 0x7fff8u) | 4u) << 5, min(__float_as_uint(root.a[j]), 1u << 24));
    }
    const unsigned om = nm == 255 ? 0u : top_bytes(c[0], c[1], c[2], c[3]);
    const unsigned ov = nv == 255 ? 0u : top_bytes(d[0], d[1], d[2], d[3]);
    st<NT>(reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.m) + i), om);
    st<NT>(reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.v) + i), ov);
    if ((threadIdx.x & 15) == 0)
      reinterpret_cast<unsigned short*>(a.scales)[i / OPT_BLOCK] = (unsigned short)(nm | (nv << 8));
  }
};

template <bool GB>
__device__ __forceinline__ double chunk_squares(const OptChunk& k);

__device__ __forceinline__ AdamwArgs shifted(AdamwArgs a, long long go) {
  a.chunks = gsh(a.chunks, go);
  a.m = gsh(reinterpret_cast<char*>(a.m), go);
  a.v = gsh(reinterpret_cast<char*>(a.v), go);
  a.scales = gsh(a.scales, go);
  a.step = gsh(a.step, go);
  a.partials = gsh(a.partials, go);
  a.norm = gsh(a.norm, go);
  a.skip = gsh(a.skip, go);
  return a;
}
// lr sqrt(1 - b2^t) / (1 - b1^t);  1 - b^t = -expm1(t log b): the product in double, so that its
// rounding does not grow with t
__device__ __forceinline__ float alpha_of(const AdamwArgs& a, int t) {
  return a.lr * sqrtf(-expm1f((float)(t * a.log_b2))) / -expm1f((float)(t * a.log_b1));
}
// factor of the scaled gradients; a norm that is not finite makes every gradient NaN
__device__ __forceinline__ float clip_of(const AdamwArgs& a, float norm) {
  const float scaled = norm * fabsf(a.grad_scale);
  return scaled <= a.clip ? 1.f : scaled < INFINITY ? a.clip / scaled : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ float norm_of(const double* partials, int n) {  // n: 1 .. OPT_MAX_GRID
  double v[OPT_MAX_GRID / TPB], s = 0.0;
#pragma unroll
  for (int j = 0; j < OPT_MAX_GRID / TPB; ++j) {  // in flight together: -0.8 us a clipped step
    const int i = threadIdx.x + j * TPB;
    v[j] = partials[i < n ? i : 0];
  }
#pragma unroll
  for (int j = 0; j < OPT_MAX_GRID / TPB; ++j) s += threadIdx.x + j * TPB < n ? v[j] : 0.0;
  return (float)sqrt(block_sum64(s));
}

// What a launch of one workgroup a piece (FULL) reads instead of working it out in each of them:
// counts the step and leaves norm, alpha, the gradients' factor and the step's number.
__global__ __launch_bounds__(TPB) void adamw_begin_kernel(AdamwArgs a, GroupArg ga) {
  a = shifted(a, goff(ga));
  if (a.skip && *a.skip) return;
  const int t = a.step[0] + 1;
  float norm = 0.f, clip = 1.f;
  if (a.clip > 0.f) {
    norm = norm_of(a.partials, a.npartials);
    clip = clip_of(a, norm);
  }
  __syncthreads();  // every wave has read the counter
  for (int i = threadIdx.x; i < OPT_MAX_GRID; i += TPB) a.step[i] = t;
  if (threadIdx.x == 0) {
    if (a.clip > 0.f) a.norm[0] = norm;
    a.norm[1] = alpha_of(a, t);
    a.norm[2] = clip;
    a.norm[3] = __int_as_float(t);
  }
}

template <int BITS, bool GB, int ROWS, bool NT, bool FULL>
__global__ __launch_bounds__(TPB) void adamw_kernel(AdamwArgs a, GroupArg ga) {
  const long long go = goff(ga);
  a = shifted(a, go);
  if (a.skip && *a.skip) {  // moments, weights and the step counter stay as they are
    if (a.hostflag && (*a.skip & ~1) && blockIdx.x == 0 && threadIdx.x == 0)  // as rmsprop_kernel
      __hip_atomic_store(a.hostflag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    return;
  }
  int t;
  Hyper h{a.b1, a.omb1, a.b2, a.omb2, 0.f, a.eps, a.grad_scale, 1.f};
  if constexpr (FULL) {
    h.alpha = a.norm[1];
    h.clip = a.norm[2];
    t = __float_as_int(a.norm[3]);
  } else {
    t = a.step[blockIdx.x] + 1;
    h.alpha = alpha_of(a, t);
    if (a.clip > 0.f) {
      float norm;
      if (a.partials) {
        norm = norm_of(a.partials, a.npartials);
      } else {  // a small table: every workgroup sums all of it
        double s = 0.0;
        for (int c = 0; c < a.nchunks; ++c) s += chunk_squares<GB>(get_chunk(a.chunks + c, go));
        norm = (float)sqrt(block_sum64(s));
      }
      if (blockIdx.x == 0 && threadIdx.x == 0) a.norm[0] = norm;
      h.clip = clip_of(a, norm);
    }
  }
  const unsigned salt = (unsigned)t * HASH_STEP;
  const int e0 = threadIdx.x * 4;
  for (int c = blockIdx.x; c < a.nchunks; c += gridDim.x) {
    const OptChunk k = get_chunk(a.chunks + c, go);
    const float lr_wd = k.flags & OPT_DECAY ? a.lr_wd : 0.f;
    const bool vec = k.flags & OPT_VEC;
    State<BITS, NT> s[ROWS];
    F4 w[ROWS], g[ROWS];
    if (vec && k.n == ROWS * TPB * 4) {
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        w[u] = ld4<NT>(k.w + e);
        g[u] = ldg4<GB, FULL && !GB>(k.g, e);
        s[u].load(a, k.base + e);
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int e = e0 + u * TPB * 4;
        s[u].step(a, k.base + e, w[u], g[u], lr_wd, h, salt);
        st4<NT>(k.w + e, w[u]);
      }
    } else {
      // the state reaches to the next multiple of 64, so whole blocks (16 lanes) take part
      const int end = (k.n + OPT_BLOCK - 1) / OPT_BLOCK * OPT_BLOCK;
      for (int e = e0; e < end; e += TPB * 4) {
        w[0] = edge_w(k.w, e, k.n, vec);
        g[0] = edge_g<GB>(k.g, e, k.n, vec);
        s[0].load(a, k.base + e);
        s[0].step(a, k.base + e, w[0], g[0], lr_wd, h, salt);
        edge_st(k.w, e, k.n, vec, w[0]);
      }
    }
  }
  if constexpr (!FULL) {
    __syncthreads();  // every wave has read the counter
    for (int i = blockIdx.x + threadIdx.x * gridDim.x; i < OPT_MAX_GRID; i += TPB * gridDim.x) a.step[i] = t;
  }
}

// Squares and sums in double: gradients below 1e-19 or above 1e19 have no fp32 squares.  Each
// workgroup sums its pieces in a fixed order.
__device__ __forceinline__ double sum4(const F4& g) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) s = fma((double)g.a[j], (double)g.a[j], s);
  return s;
}
// this thread's part of a full piece's sum
template <bool GB, int ROWS>
__device__ __forceinline__ double full_squares(const OptChunk& k) {
  double s = 0.0;
  if constexpr (GB) {
    // Converting to double costs more than reading a bf16 (120M: 72 us, this way 40).  Its square is
    // exact in fp32, so a thread's squares of this piece are summed there, unless their sum is so small or
    // large that some may have left fp32's range.
    uint4 x[ROWS / 2];
#pragma unroll
    for (int u = 0; u < ROWS / 2; ++u)
      x[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16_t*>(k.g) + threadIdx.x * 8 + u * TPB * 8);
    float f[ROWS / 2][8], q = 0.f;
#pragma unroll
    for (int u = 0; u < ROWS / 2; ++u) {
      unpack8(x[u], f[u]);
      q += ((f[u][0] * f[u][0] + f[u][1] * f[u][1]) + (f[u][2] * f[u][2] + f[u][3] * f[u][3])) +
           ((f[u][4] * f[u][4] + f[u][5] * f[u][5]) + (f[u][6] * f[u][6] + f[u][7] * f[u][7]));
    }
    if (q > 0x1p-90f && q < 0x1p100f) return (double)q;
#pragma unroll
    for (int u = 0; u < ROWS / 2; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fma((double)f[u][j], (double)f[u][j], s);
  } else {
    F4 g[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) g[u] = ldg4<GB>(k.g, threadIdx.x * 4 + u * TPB * 4);
#pragma unroll
    for (int u = 0; u < ROWS; ++u) s += sum4(g[u]);
  }
  return s;
}
template <bool GB>
__device__ __forceinline__ double chunk_squares(const OptChunk& k) {
  const bool vec = k.flags & OPT_VEC;
  if (vec && k.n == OPT_CHUNK_BIG) return full_squares<GB, OPT_CHUNK_BIG / (TPB * 4)>(k);
  if (vec && k.n == OPT_CHUNK) return full_squares<GB, OPT_CHUNK / (TPB * 4)>(k);
  double s = 0.0;
  for (int e = threadIdx.x * 4; e < k.n; e += TPB * 4) s += sum4(edge_g<GB>(k.g, e, k.n, vec));
  return s;
}

template <bool GB>
__global__ __launch_bounds__(TPB) void grad_norm_kernel(const OptChunk* chunks, int nchunks, double* partials,
                                                        GroupArg ga) {
  const long long go = goff(ga);
  chunks = gsh(chunks, go);
  partials = gsh(partials, go);
  double s = 0.0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) s += chunk_squares<GB>(get_chunk(chunks + c, go));
  s = block_sum64(s);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// The norm of a small table in one launch: a wave takes a piece at a time.
constexpr int ONE_TPB = 1024;
template <bool GB>
__global__ __launch_bounds__(ONE_TPB) void grad_norm_one_kernel(const OptChunk* chunks, int nchunks, float* out) {
  __shared__ double part[ONE_TPB / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = 0.0;
  for (int c = wave; c < nchunks; c += ONE_TPB / 64) {
    const OptChunk k = get_chunk(chunks + c, 0);
    const bool vec = k.flags & OPT_VEC;
    for (int e = lane * 4; e < k.n; e += 1024) {
      F4 g[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = edge_g<GB>(k.g, e + j * 256, k.n, vec);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += sum4(g[j]);
    }
  }
  s = wave_sum64(s);
  if (lane == 0) part[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < ONE_TPB / 64; ++i) s += part[i];
    *out = (float)sqrt(s);
  }
}

__global__ __launch_bounds__(TPB) void norm_of_partials_kernel(const double* partials, int n, float* out) {
  const float norm = norm_of(partials, n);
  if (threadIdx.x == 0) *out = norm;
}

// A thread takes 8 codes of each kind: in bf16 their values are one 16-byte store.
template <bool OB, bool NT>
__global__ __launch_bounds__(TPB) void adamw_decode_kernel(const unsigned char* m, const unsigned char* v,
                                                           const unsigned char* scales, long long n8, void* om,
                                                           void* ov) {
  typedef unsigned vu2 __attribute__((ext_vector_type(2)));
  typedef unsigned vu4 __attribute__((ext_vector_type(4)));
  const long long i = blockIdx.x * (long long)TPB + threadIdx.x;
  if (i < n8) {
    const vu2 m8 = ld<NT>(reinterpret_cast<const vu2*>(m) + i), v8 = ld<NT>(reinterpret_cast<const vu2*>(v) + i);
    const unsigned sc = reinterpret_cast<const unsigned short*>(scales)[i / (OPT_BLOCK / 8)];
    const int sm = sc & 255, sv = sc >> 8;
    const float nan = __uint_as_float(0x7fc00000u);
    F4 x[2], y[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      x[k] = F4{{m_value<0>(m8[k], sm), m_value<1>(m8[k], sm), m_value<2>(m8[k], sm), m_value<3>(m8[k], sm)}};
      y[k] = F4{{root_value<0>(v8[k], sv), root_value<1>(v8[k], sv), root_value<2>(v8[k], sv), root_value<3>(v8[k], sv)}};
      if (sm == 255) x[k] = F4{{nan, nan, nan, nan}};
      if (sv == 255) y[k] = F4{{nan, nan, nan, nan}};
    }
    if constexpr (OB) {  // exact: at most 5 significant bits
      st<NT>(reinterpret_cast<vu4*>(om) + i, vu4{pack2bf(x[0].a[0], x[0].a[1]), pack2bf(x[0].a[2], x[0].a[3]),
                                                 pack2bf(x[1].a[0], x[1].a[1]), pack2bf(x[1].a[2], x[1].a[3])});
      st<NT>(reinterpret_cast<vu4*>(ov) + i, vu4{pack2bf(y[0].a[0], y[0].a[1]), pack2bf(y[0].a[2], y[0].a[3]),
                                                 pack2bf(y[1].a[0], y[1].a[1]), pack2bf(y[1].a[2], y[1].a[3])});
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        st4<NT>(reinterpret_cast<float*>(om) + 8 * i + 4 * k, x[k]);
        st4<NT>(reinterpret_cast<float*>(ov) + 8 * i + 4 * k, y[k]);
      }
    }
  }
}

}  // namespace

namespace {
// us, cold (three sets of tensors in turn), one MI355X:
//   cached / past the caches (NT), 4096 pieces: fp32 gradients, 32-bit states: 7M weights 35.8 / 33.1, 18M
//   100.7 / 80.6, 120M 655 / 611; 8-bit states: 7M 22.2 / 22.9, 18M 62.2 / 50.8, 120M 385 / 355.  So NT is
//   for weights and states that do not stay in the 256 MB of the last cache anyway (OPT_NT_BYTES).  Gradients
//   have just been written and are read through it (18M: 80.6 / 89.8 with them past it), but fp32 ones
//   of the largest tables (120M: 611 / 607).
//   1024 workgroups that take pieces in turn / a workgroup for each piece (FULL): 18M 80.8 / 78.2, 35M 169 / 161,
//   70M 345 / 324, 120M 596 / 561; 8 bits: 35M 103 / 98, 120M 367 / 324.  FULL costs a launch (the step
//   counter has one word for each of 1024 workgroups): from 8 pieces each on.
template <int BITS, bool GB>
void launch_adamw(const AdamwArgs& a, hipStream_t st) {
  const dim3 grid = ggrid(opt_grid(a.nchunks));
  constexpr int R = OPT_CHUNK / (TPB * 4), RB = OPT_CHUNK_BIG / (TPB * 4);
  if (a.chunk == OPT_CHUNK) {
    hipLaunchKernelGGL((adamw_kernel<BITS, GB, R, false, false>), grid, dim3(TPB), 0, st, a, garg());
  } else if ((long long)a.nchunks * a.chunk * (BITS == 8 ? 12 : 24) < OPT_NT_BYTES) {
    hipLaunchKernelGGL((adamw_kernel<BITS, GB, RB, false, false>), grid, dim3(TPB), 0, st, a, garg());
  } else if (a.nchunks < 8 * OPT_MAX_GRID) {
    hipLaunchKernelGGL((adamw_kernel<BITS, GB, RB, true, false>), grid, dim3(TPB), 0, st, a, garg());
  } else {
    hipLaunchKernelGGL(adamw_begin_kernel, ggrid(1), dim3(TPB), 0, st, a, garg());
    hipLaunchKernelGGL((adamw_kernel<BITS, GB, RB, true, true>), ggrid(a.nchunks), dim3(TPB), 0, st, a, garg());
  }
}
}  // namespace

hipError_t adamw(const AdamwArgs& a, int bits, int g_bf16, hipStream_t st) {
  if ((bits != 8 && bits != 32) || (a.chunk != OPT_CHUNK && a.chunk != OPT_CHUNK_BIG) || !a.step || a.nchunks < 0 ||
      !a.norm || (a.nchunks && !(a.chunks && a.m && a.v)) || (bits == 8 && a.nchunks && !a.scales))
    return hipErrorInvalidValue;
  if (a.clip > 0.f && (a.partials ? a.npartials < 1 || a.npartials > OPT_MAX_GRID : a.nchunks > OPT_OWN_SUM))
    return hipErrorInvalidValue;
  if (bits == 8) {
    if (g_bf16) launch_adamw<8, true>(a, st);
    else launch_adamw<8, false>(a, st);
  } else {
    if (g_bf16) launch_adamw<32, true>(a, st);
    else launch_adamw<32, false>(a, st);
  }
  return hipGetLastError();
}

hipError_t grad_norm_partials(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, hipStream_t st) {
  if (nchunks < 0 || (nchunks && !chunks) || !partials) return hipErrorInvalidValue;
  const dim3 grid = ggrid(opt_grid(nchunks));
  if (g_bf16) hipLaunchKernelGGL(grad_norm_kernel<true>, grid, dim3(TPB), 0, st, chunks, nchunks, partials, garg());
  else hipLaunchKernelGGL(grad_norm_kernel<false>, grid, dim3(TPB), 0, st, chunks, nchunks, partials, garg());
  return hipGetLastError();
}

hipError_t grad_norm(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, float* out, hipStream_t st) {
  if (nchunks < 0 || (nchunks && !chunks) || (nchunks > OPT_NORM_ONE && !partials) || !out) return hipErrorInvalidValue;
  if (nchunks <= OPT_NORM_ONE) {
    if (g_bf16) hipLaunchKernelGGL(grad_norm_one_kernel<true>, dim3(1), dim3(ONE_TPB), 0, st, chunks, nchunks, out);
    else hipLaunchKernelGGL(grad_norm_one_kernel<false>, dim3(1), dim3(ONE_TPB), 0, st, chunks, nchunks, out);
    return hipGetLastError();
  }
  const int grid = opt_grid(nchunks);
  const GroupArg alone{0, 1, 0};
  if (g_bf16) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3(grid), dim3(TPB), 0, st, chunks, nchunks, partials, alone);
  else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3(grid), dim3(TPB), 0, st, chunks, nchunks, partials, alone);
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
  const long long n8 = n / 8, blocks = (n8 + TPB - 1) / TPB;
  const dim3 grid((unsigned)blocks);
  const bool nt = n * (out_bf16 ? 6 : 10) >= OPT_NT_BYTES;
  if (out_bf16) {
    if (nt) hipLaunchKernelGGL((adamw_decode_kernel<true, true>), grid, dim3(TPB), 0, st, m, v, scales, n8, om, ov);
    else hipLaunchKernelGGL((adamw_decode_kernel<true, false>), grid, dim3(TPB), 0, st, m, v, scales, n8, om, ov);
  } else {
    if (nt) hipLaunchKernelGGL((adamw_decode_kernel<false, true>), grid, dim3(TPB), 0, st, m, v, scales, n8, om, ov);
    else hipLaunchKernelGGL((adamw_decode_kernel<false, false>), grid, dim3(TPB), 0, st, m, v, scales, n8, om, ov);
  }
  return hipGetLastError();
}

}  // namespace idc
