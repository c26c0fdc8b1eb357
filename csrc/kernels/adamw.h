#pragma once
#include "common.h"

namespace idc {

// One piece of one tensor of a multi-tensor optimizer launch (ops/optim.py TensorTable).
struct OptChunk {
  float* w;          // weights of the piece (null in a table that only serves the norm)
  const void* g;     // gradients, fp32 or bf16
  long long base;    // the piece's place in the flat state: a multiple of 64
  int n;             // elements, 1 .. the table's chunk size
  int flags;         // bit 0: weight decay; bit 1: w and g begin at multiples of 16 bytes
};
// Elements a workgroup takes at a time: OPT_CHUNK, and OPT_CHUNK_BIG in a table that has at least
// OPT_MAX_GRID pieces of that size.  us for fp32 gradients, 32-bit states, 2048 / 4096: 2.2M weights 11.4 /
// 11.8, 7M 36.0 / 35.8, 40M 225 / 216, 120M 669 / 655.
constexpr int OPT_CHUNK = 2048, OPT_CHUNK_BIG = 4096;
constexpr long long OPT_NT_BYTES = 128ll << 20;  // what is read and written from here on goes past the caches
constexpr int OPT_MAX_GRID = 1024;    // workgroups of a launch, copies of the step counter, partial sums
// Pieces that a clipped step's workgroups all sum by themselves: 8 take 6.1 us, with a launch ahead 6.8.
constexpr int OPT_OWN_SUM = 8;
// Pieces that grad_norm leaves to one workgroup: 32 take 4.8 us, two launches 5.3 and a workspace; 48 6.5.
constexpr int OPT_NORM_ONE = 32;
constexpr int OPT_DECAY = 1, OPT_VEC = 2;
constexpr int OPT_BLOCK = 64;         // elements that share a scale in an 8-bit state

struct AdamwArgs {
  const OptChunk* chunks;
  void* m;                  // first moments: fp32, or 8-bit codes
  void* v;                  // second moments: fp32, or 8-bit codes of their roots
  unsigned char* scales;    // 8-bit states: [block][2] scale bytes (first moment, root)
  int* step;                // [OPT_MAX_GRID] copies of the steps done
  const double* partials;   // sums of squared gradients (grad_norm_partials); null with clipping: at
                            // most OPT_OWN_SUM pieces, the step sums them itself
  float* norm;              // [4] the global norm, written when there is clipping; work space
  const int* skip;          // nullable guard word: not zero = this step changes nothing
  int* hostflag;            // nullable pinned host word (rmsprop's)
  double log_b1, log_b2;    // natural logarithms of beta_1, beta_2 (-inf for 0)
  float b1, omb1, b2, omb2; // betas, and 1 - beta rounded from double
  float lr, eps, lr_wd;     // lr_wd = learning rate * weight decay
  float grad_scale, clip;   // clip: largest norm of the scaled gradients (0: no clipping)
  int nchunks, npartials;
  int chunk, pad;           // the table's chunk size
};

inline int opt_grid(int nchunks) { return nchunks < 1 ? 1 : nchunks > OPT_MAX_GRID ? OPT_MAX_GRID : nchunks; }

hipError_t adamw(const AdamwArgs& a, int bits, int g_bf16, hipStream_t st);
hipError_t adamw_decode(const unsigned char* m, const unsigned char* v, const unsigned char* scales, long long n,
                        void* om, void* ov, int out_bf16, hipStream_t st);
hipError_t grad_norm_partials(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, hipStream_t st);
hipError_t grad_norm(const OptChunk* chunks, int nchunks, int g_bf16, double* partials, float* out, hipStream_t st);

}  // namespace idc
