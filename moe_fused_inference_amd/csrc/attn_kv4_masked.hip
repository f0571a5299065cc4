// attn_kv4_masked.hip -- the kernels of attn_kv4_few.h with masks (windows, trees).
#include "attn_kv4_few.h"

int mxa::attn_few_masked(const Args& a, int q_dtype, const Plan& p, int D, bool much, hipStream_t st) {
    return launch_few<true>(a, q_dtype, p, D, much, st);
}
