// Host side of the split form of the biased attention for few queries (token_attention.hip).
#pragma once
#include <stdint.h>

namespace mivae {

struct BiasedArgs;

// floats of the partials' buffer, 0 where the keys are not split
int64_t token_attention_floats(int64_t B, int64_t Sq, int64_t Sk, int64_t heads, int64_t kv, int64_t d);
// launches; the caller has checked the arguments and looks at the launch status
void token_attention(const BiasedArgs& a, float* scratch, int dtype, void* stream);

// out (and lse, out_lo) from `splits` partials per row of (b, head, row): [row][split][d + 4] of O, max, sum
void token_attention_join(const BiasedArgs& a, float* part, int splits, int dtype, void* stream);

}  // namespace mivae
