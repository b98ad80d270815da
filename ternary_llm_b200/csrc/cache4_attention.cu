// Attention over the 4-bit key/value cache for sequences of different lengths: which kernel takes a call.
#include "cache4.cuh"
#include "cache4_work.cuh"

namespace tllm {

// Rows of a key/value head go 16 at once through mma.sync up to 32 of them, and while a tile of 16 an SM takes the call and stays in one CTA; behind
// that 128 or 256 at once through tcgen05.  Both sides, us, 32 heads over 8, caches beyond L2 in turn: of 128, one sequence of 64 tokens behind 700
// 12.5 / 16.4, of 40 behind 1200 15.8 / 19.5, behind 1800 23.0 / 19.8, of 64 behind 6000 51.8 / 26.1, 14 of 9 (336 tiles) behind 300 24.1 / 11.9; of 64,
// one of 64 behind 2400 about equal, behind 6000 35.5 / 22.0.  Up to 32 rows: 14 of 4 behind 6000 47.6 / 77.2, 6 of 5 behind 2500 27.3 / 24.2, of 64
// 32.9 / 64.1 and 20.4 / 21.2.
static bool takes_step(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    const long long rows = (long long)new_rows(c, tokens, max_new) * (heads / c.kv_heads);
    const long long tiles = (rows + 15) / 16 * c.batch * c.kv_heads, len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    return rows <= 32 || (tiles <= 148 && len <= kStepWhole / c.dim);
}

// The way of a call: few rows, or prompts.  More units than the first can count, which a number of new rows far below the real one asks for, are
// prompts of unknown length.
struct Way {
    bool few;
    StepPlan step;
    PromptPlan prompt;
};
static Way way_of(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    Way w = {};
    const int len = max_len > 0 && max_len < c.rows ? max_len : c.rows;
    if (takes_step(c, tokens, heads, max_new, max_len)) {
        w.step = step_plan(c, tokens, heads, max_new, max_len);
        w.few = work_fits(c, tokens, heads, len, w.step.rows, kStepChunk, w.step.whole);
        if (!w.few) max_new = 0;
    }
    if (!w.few) w.prompt = prompt_plan(c, tokens, heads, max_new, max_len);
    return w;
}

size_t cache4_workspace(const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    if (tokens == 0 || c.batch == 0) return 0;
    const Way w = way_of(c, tokens, heads, max_new, max_len);
    return w.few ? w.step.bytes : w.prompt.bytes;
}

template <typename T>
int launch_cache4_attention(const Cache4Call& a, Rows<const T> q, Rows<T> out, cudaStream_t stream)
{
    if (a.s.tokens == 0 || a.s.batch == 0) return TLLM_OK;
    const Way w = way_of(a.c, a.s.tokens, a.heads, a.max_new, a.max_len);
    return w.few ? launch_cache4_step<T>(a, q, out, w.step, stream) : launch_cache4_prompt<T>(a, q, out, w.prompt, stream);
}

template int launch_cache4_attention<half>(const Cache4Call&, Rows<const half>, Rows<half>, cudaStream_t);
template int launch_cache4_attention<bf16>(const Cache4Call&, Rows<const bf16>, Rows<bf16>, cudaStream_t);

}  // namespace tllm
