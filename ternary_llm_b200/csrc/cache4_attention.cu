// Attention over the 4-bit key/value cache for sequences of different lengths: which kernel takes a call.
#include "cache4.cuh"
#include "cache4_work.cuh"

namespace tllm {

// Rows of a key/value head go 16 at once through mma.sync up to 32 of them, and while one tile of 16 a SM takes the call; behind that 256 at once
// through tcgen05.  Both sides, us, 32 heads over 8: of 64, 6 sequences of 5 tokens behind 3000 21.1 / 27.4, 24 of 8 behind 1000 30.4 / 35.2; of
// 128, 24 of 8 behind 3000 75 / 83, one of 16 behind 3000 18.6 / 23.6, one of 32 23.4 / 25.0 (64 tiles), 6 of 16 45.7 / 33.8 (192 tiles), 6 of 32
// behind 200 22.1 / 15.5.
static bool takes_step(const Cache4& c, int tokens, int heads, int max_new)
{
    const long long rows = (long long)(max_new > 0 && max_new < tokens ? max_new : tokens) * (heads / c.kv_heads);
    return rows <= 32 || (rows + 15) / 16 * c.batch * c.kv_heads <= 148;
}

size_t cache4_workspace(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    if (tokens == 0 || c.batch == 0) return 0;
    return takes_step(c, tokens, heads, max_new) ? step_plan(c, tokens, heads, max_new, max_len).bytes : prompt_plan(c, tokens, heads, max_new, max_len).bytes;
}

template <typename T>
int launch_cache4_attention(const Cache4Call& a, Rows<const T> q, Rows<T> out, cudaStream_t stream)
{
    if (a.s.tokens == 0 || a.s.batch == 0) return TLLM_OK;
    const bool step = takes_step(a.c, a.s.tokens, a.heads, a.max_new);
    if (!work_fits(a, step ? 4 : kPromptRows, step ? kStepChunk : kPromptChunk))
        return fail(TLLM_ERR_SIZE, "cache4_attention: %d rows of %d heads over %d positions", a.s.tokens, a.heads, a.c.rows);
    if (step)
        return launch_cache4_step<T>(a, q, out, step_plan(a.c, a.s.tokens, a.heads, a.max_new, a.max_len), stream);
    return launch_cache4_prompt<T>(a, q, out, prompt_plan(a.c, a.s.tokens, a.heads, a.max_new, a.max_len), stream);
}

template int launch_cache4_attention<half>(const Cache4Call&, Rows<const half>, Rows<half>, cudaStream_t);
template int launch_cache4_attention<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, cudaStream_t);

}  // namespace tllm
