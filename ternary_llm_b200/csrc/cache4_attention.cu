// Attention over the 4-bit key/value cache for sequences of different lengths: which kernel takes a call.
#include "cache4.cuh"
#include "cache4_work.cuh"

namespace tllm {

// Rows of a key/value head go 16 at once through mma.sync up to 32 of them, and while a tile of 16 a SM takes the call and its positions are few;
// behind that 128 or 256 at once through tcgen05.  Both sides, us, 32 heads over 8: of 64, 14 sequences of 4 tokens behind 6000 31 / 73, one of 64
// behind 2500 23.7 / 24.6, behind 6000 34 / 28; of 128, one of 40 (80 tiles) behind 2500 24 / 29, behind 6000 35 / 33, one of 64 (128) behind
// 300 9.3 / 14.3, behind 6000 49 / 34, 14 of 9 (336) behind 300 22 / 14, behind 2500 60 / 47.
static bool takes_step(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    const long long rows = (long long)new_rows(c, tokens, max_new) * (heads / c.kv_heads);
    const long long tiles = (rows + 15) / 16 * c.batch * c.kv_heads, len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    return rows <= 32 || (tiles <= 148 && (len <= kStepWhole / c.dim || tiles * len <= 40000000 / c.dim));
}

size_t cache4_workspace(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    if (tokens == 0 || c.batch == 0) return 0;
    return takes_step(c, tokens, heads, max_new, max_len) ? step_plan(c, tokens, heads, max_new, max_len).bytes : prompt_plan(c, tokens, heads, max_new, max_len).bytes;
}

template <typename T>
int launch_cache4_attention(const Cache4Call& a, Rows<const T> q, Rows<T> out, cudaStream_t stream)
{
    if (a.s.tokens == 0 || a.s.batch == 0) return TLLM_OK;
    const bool step = takes_step(a.c, a.s.tokens, a.heads, a.max_new, a.max_len);
    if (!work_fits(a, step ? 4 : 128, step ? kStepChunk : kPromptChunk))
        return fail(TLLM_ERR_SIZE, "cache4_attention: %d rows of %d heads over %d positions", a.s.tokens, a.heads, a.c.rows);
    if (step)
        return launch_cache4_step<T>(a, q, out, step_plan(a.c, a.s.tokens, a.heads, a.max_new, a.max_len), stream);
    return launch_cache4_prompt<T>(a, q, out, prompt_plan(a.c, a.s.tokens, a.heads, a.max_new, a.max_len), stream);
}

template int launch_cache4_attention<half>(const Cache4Call&, Rows<const half>, Rows<half>, cudaStream_t);
template int launch_cache4_attention<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, cudaStream_t);

}  // namespace tllm
