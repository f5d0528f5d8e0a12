// Attention within sequences: what the launchers of attention_fwd.cu and attention_bwd.cu take.
#pragma once
#include <cuda_runtime.h>

namespace tn {

// One operand, bf16: element (b, t, h, d) at p[b * sb + t * st + h * sh + d].  Packed sequences have b = 0 and t over all tokens.
struct AttnOperand {
  void* p;
  long long sb, st, sh;
};

// Where the sequences of queries or of keys lie.  Padded (off null): sequence n is the first len[n] rows (len null: all T) of b = n.
// Packed: rows off[n] to off[n + 1] of T.  Values outside the operand are cut to it.
struct AttnRows {
  const int* off;
  const int* len;
  int T;
};

struct AttnArgs {
  int B, H, G, D;              // sequences, query heads, key heads (H a multiple of G), columns (a multiple of 8, up to 128)
  AttnRows rq, rk;
  AttnOperand q, k, v, o;      // o: written forward, read backward
  AttnOperand rest;            // what rounding took off o, rounded itself (p null: not kept); the backward pass sums do (o + rest)
  float* lse;                  // [H][rows of q] log2 of the sums of exponentials, +inf where a row sees nothing; forward: may be null
  float scale;                 // of the products, above 0
  float cap;                   // 0: none
  const float* slopes;         // [H] or null
  const int* prefix;           // [B] or null
  int causal;
  int newest;                  // every query stands at the last key (not with causal)
  float step;                  // of a query's place to the next one's: 0 where newest, else 1
  // backward
  AttnOperand go, gq, gk, gv;
  float* delta;                // [H][rows of q] workspace
  int* status;
};

const char* launch_attention_fwd(const AttnArgs& a, cudaStream_t st);
// Few queries, padded: whether launch_attention_few takes the call (it is asked first), and the fp32 values of workspace that it wants then.
bool attention_few_takes(const AttnArgs& a);
long long attention_few_floats(const AttnArgs& a);
const char* launch_attention_few(const AttnArgs& a, float* work, cudaStream_t st);
// Short sequences of up to 64 columns: whether the warp-per-tile kernels take the call.  launch_attention_bwd asks by itself.
bool attention_short_takes(const AttnArgs& a, bool backward);
const char* launch_attention_short_fwd(const AttnArgs& a, cudaStream_t st);
const char* launch_attention_short_bwd(const AttnArgs& a, cudaStream_t st);
const char* launch_attention_bwd(const AttnArgs& a, cudaStream_t st);

}  // namespace tn
