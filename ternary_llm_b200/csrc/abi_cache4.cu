// extern "C" entry points of the 4-bit key/value cache (include/tllm_b200_cache4.h): argument checks
// and dispatch to rotary.cu, cache4_rows.cu and cache4_attention.cu.
#include <climits>
#include <cmath>
#include <utility>

#include "cache4.cuh"

using namespace tllm;

namespace {

constexpr int kMostHeads = 4096, kMostTokens = INT_MAX - 16;

inline bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
inline size_t type_size(int type) { return type == TLLM_FP32 ? 4 : 2; }

int check_type(const char* fn, int type, bool fp32)
{
    if (type != TLLM_FP16 && type != TLLM_BF16 && !(fp32 && type == TLLM_FP32)) return fail(TLLM_ERR_SHAPE, "%s: activation type %d", fn, type);
    return TLLM_OK;
}

int check_rows(const char* fn, const char* name, const tllm_b200_heads* x, int type, int tokens, int heads, int dim)
{
    if (!x || (!x->p && tokens > 0)) return fail(TLLM_ERR_NULL, "%s: %s is null", fn, name);
    const long long width = (long long)heads * dim;
    if (x->ld < (tokens > 1 ? width : 0) || x->ld > (1ll << 40)) return fail(TLLM_ERR_SHAPE, "%s: rows of %s are %lld elements apart, %lld wide", fn, name, x->ld, width);
    if (misaligned(x->p, 16) || x->ld * type_size(type) % 16) return fail(TLLM_ERR_ALIGN, "%s: rows of %s must lie on 16-byte boundaries", fn, name);
    return TLLM_OK;
}

// Rows of an output, and those of an input or another output: the same where that is allowed, or apart.
int check_apart(const char* fn, const char* name, const tllm_b200_heads* x, int x_heads, const tllm_b200_heads* y, int y_heads, int type, int tokens, int dim,
                bool same)
{
    if (tokens == 0 || (same && x->p == y->p && (x->ld == y->ld || tokens == 1))) return TLLM_OK;
    if (x->p > y->p) std::swap(x, y), std::swap(x_heads, y_heads);
    const size_t one = type_size(type), off = reinterpret_cast<uintptr_t>(y->p) - reinterpret_cast<uintptr_t>(x->p), step = (size_t)x->ld * one;
    const size_t width = (size_t)x_heads * dim * one, other = (size_t)y_heads * dim * one;
    if (off >= (size_t)(tokens - 1) * step + width) return TLLM_OK;
    // rows between rows of the other, equally far apart
    if (tokens > 1 && x->ld == y->ld && off % step >= width && off % step + other <= step) return TLLM_OK;
    return fail(TLLM_ERR_SHAPE, "%s: %s overlaps an output", fn, name);
}

int check_table(const char* fn, const tllm_b200_rotary_table* t, int dim, int inverse, Rotary* r)
{
    *r = Rotary{nullptr, 0, 0, 1.f, inverse};
    if (!t) return TLLM_OK;
    if (!t->turns) return fail(TLLM_ERR_NULL, "%s: the table is null", fn);
    if (t->rot_dim < 2 || t->rot_dim % 2 || t->rot_dim > dim) return fail(TLLM_ERR_SHAPE, "%s: %d of %d entries of a head turn", fn, t->rot_dim, dim);
    if (misaligned(t->turns, 8)) return fail(TLLM_ERR_ALIGN, "%s: the table must be 8-byte aligned", fn);
    if (!std::isfinite(t->amplitude)) return fail(TLLM_ERR_SHAPE, "%s: amplitude %g", fn, t->amplitude);
    *r = Rotary{t->turns, t->rot_dim, t->half_layout != 0, t->amplitude, inverse};
    return TLLM_OK;
}

int check_cache(const char* fn, const tllm_b200_cache4* c, Cache4* v)
{
    if (!c || (c->batch != 0 && (!c->k_codes || !c->k_params || !c->v_codes || !c->v_params))) return fail(TLLM_ERR_NULL, "%s: the cache is null", fn);
    if (c->batch < 0 || c->kv_heads < 1 || c->rows < 1 || (c->dim != 64 && c->dim != 128))
        return fail(TLLM_ERR_SHAPE, "%s: cache of batch=%d kv_heads=%d rows=%d dim=%d (64 or 128)", fn, c->batch, c->kv_heads, c->rows, c->dim);
    if (misaligned(c->k_codes, 16) || misaligned(c->k_params, 16) || misaligned(c->v_codes, 16) || misaligned(c->v_params, 16))
        return fail(TLLM_ERR_ALIGN, "%s: the cache's arrays must be 16-byte aligned", fn);
    *v = Cache4{(uint8_t*)c->k_codes, (uint8_t*)c->v_codes, (half2*)c->k_params, (half2*)c->v_params, c->batch, c->kv_heads, c->rows, c->dim};
    return TLLM_OK;
}

int check_seqs(const char* fn, const int* first, const int* lens, int tokens, const Cache4& c, Seqs* s)
{
    if (c.batch > 0 && (!first || !lens)) return fail(TLLM_ERR_NULL, "%s: first or lens is null", fn);
    if (tokens < 0 || tokens > kMostTokens) return fail(TLLM_ERR_SHAPE, "%s: tokens=%d", fn, tokens);
    if (misaligned(first, 4) || misaligned(lens, 4)) return fail(TLLM_ERR_ALIGN, "%s: first and lens must be 4-byte aligned", fn);
    *s = Seqs{first, lens, c.batch, tokens, c.rows, nullptr};
    return TLLM_OK;
}

int error_flag(Seqs* s)
{
    s->err = device_error_flag();
    return s->err ? TLLM_OK : fail(TLLM_ERR_LAUNCH, "device scratch unavailable");
}

template <typename T> Rows<const T> in(const tllm_b200_heads* x) { return x ? Rows<const T>{(const T*)x->p, x->ld} : Rows<const T>{nullptr, 0}; }
template <typename T> Rows<T> out(const tllm_b200_heads* x) { return x ? Rows<T>{(T*)x->p, x->ld} : Rows<T>{nullptr, 0}; }

inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int tllm_b200_rotary(int type, const tllm_b200_rotary_table* table, const int* positions, int tokens, const tllm_b200_heads* q,
                     const tllm_b200_heads* q_out, int heads, const tllm_b200_heads* k, const tllm_b200_heads* k_out, int kv_heads, int dim,
                     int inverse, void* stream)
{
    const char* fn = "rotary";
    if (!table || (!positions && tokens > 0)) return fail(TLLM_ERR_NULL, "rotary: null pointer");
    int st = check_type(fn, type, true);
    if (st) return st;
    if (tokens < 0 || tokens > kMostTokens || heads < 1 || kv_heads < 0 || heads > kMostHeads || kv_heads > kMostHeads || dim < 4 || dim > 512 || dim * type_size(type) % 16)
        return fail(TLLM_ERR_SHAPE, "rotary: tokens=%d heads=%d/%d dim=%d", tokens, heads, kv_heads, dim);
    if ((k != nullptr) != (kv_heads > 0) || (k != nullptr) != (k_out != nullptr)) return fail(TLLM_ERR_NULL, "rotary: k, k_out and kv_heads go together");
    Rotary r;
    if ((st = check_table(fn, table, dim, inverse != 0, &r)) || (st = check_rows(fn, "q", q, type, tokens, heads, dim)) ||
        (st = check_rows(fn, "q_out", q_out, type, tokens, heads, dim)) || (st = check_apart(fn, "q", q, heads, q_out, heads, type, tokens, dim, true)))
        return st;
    if (k && ((st = check_rows(fn, "k", k, type, tokens, kv_heads, dim)) || (st = check_rows(fn, "k_out", k_out, type, tokens, kv_heads, dim)) ||
              (st = check_apart(fn, "k", k, kv_heads, k_out, kv_heads, type, tokens, dim, true)) ||
              (st = check_apart(fn, "k", k, kv_heads, q_out, heads, type, tokens, dim, false)) ||
              (st = check_apart(fn, "q", q, heads, k_out, kv_heads, type, tokens, dim, false)) ||
              (st = check_apart(fn, "k_out", k_out, kv_heads, q_out, heads, type, tokens, dim, false))))
        return st;
    if (misaligned(positions, 4)) return fail(TLLM_ERR_ALIGN, "rotary: positions must be 4-byte aligned");
    if ((st = check_device())) return st;
    if (type == TLLM_FP16)
        return launch_rotary<half>(r, positions, tokens, in<half>(q), out<half>(q_out), heads, in<half>(k), out<half>(k_out), kv_heads, dim, S(stream));
    if (type == TLLM_BF16)
        return launch_rotary<bf16>(r, positions, tokens, in<bf16>(q), out<bf16>(q_out), heads, in<bf16>(k), out<bf16>(k_out), kv_heads, dim, S(stream));
    return launch_rotary<float>(r, positions, tokens, in<float>(q), out<float>(q_out), heads, in<float>(k), out<float>(k_out), kv_heads, dim, S(stream));
}

int tllm_b200_cache4_append(const tllm_b200_cache4* cache, int type, const tllm_b200_rotary_table* table, const int* first, const int* lens,
                            int tokens, const tllm_b200_heads* q, const tllm_b200_heads* q_out, int heads, const tllm_b200_heads* k,
                            const tllm_b200_heads* v, void* stream)
{
    const char* fn = "cache4_append";
    Cache4 c;
    Seqs s;
    Rotary r;
    int st;
    if ((st = check_type(fn, type, false)) || (st = check_cache(fn, cache, &c)) || (st = check_seqs(fn, first, lens, tokens, c, &s)) ||
        (st = check_table(fn, table, c.dim, 0, &r)) || (st = check_rows(fn, "k", k, type, tokens, c.kv_heads, c.dim)) ||
        (st = check_rows(fn, "v", v, type, tokens, c.kv_heads, c.dim)))
        return st;
    if (heads < 0 || heads > kMostHeads || c.kv_heads > kMostHeads) return fail(TLLM_ERR_SHAPE, "cache4_append: heads=%d/%d", heads, c.kv_heads);
    if ((q != nullptr) != (heads > 0) || (q != nullptr) != (q_out != nullptr)) return fail(TLLM_ERR_NULL, "cache4_append: q, q_out and heads go together");
    if (q && ((st = check_rows(fn, "q", q, type, tokens, heads, c.dim)) || (st = check_rows(fn, "q_out", q_out, type, tokens, heads, c.dim)) ||
              (st = check_apart(fn, "q", q, heads, q_out, heads, type, c.batch ? tokens : 0, c.dim, true)) ||
              (st = check_apart(fn, "k", k, c.kv_heads, q_out, heads, type, c.batch ? tokens : 0, c.dim, false)) ||
              (st = check_apart(fn, "v", v, c.kv_heads, q_out, heads, type, c.batch ? tokens : 0, c.dim, false))))
        return st;
    if ((st = check_device()) || (st = error_flag(&s))) return st;
    if (type == TLLM_FP16) return launch_cache4_append<half>(c, r, s, in<half>(q), out<half>(q_out), heads, in<half>(k), in<half>(v), S(stream));
    return launch_cache4_append<bf16>(c, r, s, in<bf16>(q), out<bf16>(q_out), heads, in<bf16>(k), in<bf16>(v), S(stream));
}

int tllm_b200_cache4_read(const tllm_b200_cache4* cache, int type, const int* first, const int* lens, int tokens, const tllm_b200_heads* k,
                          const tllm_b200_heads* v, void* stream)
{
    const char* fn = "cache4_read";
    Cache4 c;
    Seqs s;
    int st;
    if ((st = check_type(fn, type, true)) || (st = check_cache(fn, cache, &c)) || (st = check_seqs(fn, first, lens, tokens, c, &s))) return st;
    if (!k && !v) return fail(TLLM_ERR_NULL, "cache4_read: neither k nor v");
    if (c.kv_heads > kMostHeads) return fail(TLLM_ERR_SHAPE, "cache4_read: heads=%d", c.kv_heads);
    if ((k && (st = check_rows(fn, "k", k, type, tokens, c.kv_heads, c.dim))) || (v && (st = check_rows(fn, "v", v, type, tokens, c.kv_heads, c.dim))) ||
        (k && v && (st = check_apart(fn, "k", k, c.kv_heads, v, c.kv_heads, type, c.batch ? tokens : 0, c.dim, false))))
        return st;
    if ((st = check_device()) || (st = error_flag(&s))) return st;
    if (type == TLLM_FP16) return launch_cache4_read<half>(c, s, out<half>(k), out<half>(v), S(stream));
    if (type == TLLM_BF16) return launch_cache4_read<bf16>(c, s, out<bf16>(k), out<bf16>(v), S(stream));
    return launch_cache4_read<float>(c, s, out<float>(k), out<float>(v), S(stream));
}

static int check_heads(const char* fn, const Cache4& c, int tokens, int heads, int max_new, int max_len)
{
    if (heads < 1 || heads > kMostHeads || heads % c.kv_heads) return fail(TLLM_ERR_SHAPE, "%s: %d query heads over %d", fn, heads, c.kv_heads);
    if ((long long)tokens * heads > INT_MAX) return fail(TLLM_ERR_SHAPE, "%s: %d rows of %d heads", fn, tokens, heads);
    if (max_new < 0 || max_len < 0) return fail(TLLM_ERR_SHAPE, "%s: max_new=%d max_len=%d", fn, max_new, max_len);
    return TLLM_OK;
}

int tllm_b200_cache4_workspace(const tllm_b200_cache4* cache, int tokens, int heads, int max_new, int max_len, size_t* bytes)
{
    const char* fn = "cache4_workspace";
    Cache4 c;
    int st;
    if (!bytes) return fail(TLLM_ERR_NULL, "cache4_workspace: null pointer");
    if ((st = check_cache(fn, cache, &c)) || (st = check_heads(fn, c, tokens, heads, max_new, max_len))) return st;
    if (tokens < 0) return fail(TLLM_ERR_SHAPE, "cache4_workspace: tokens=%d", tokens);
    *bytes = cache4_workspace(c, tokens, heads, max_new, max_len);
    return TLLM_OK;
}

int tllm_b200_cache4_attention(const tllm_b200_cache4* cache, int type, const int* first, const int* lens, int tokens,
                               const tllm_b200_heads* q, const tllm_b200_heads* out_rows, int heads, float scale, int max_new, int max_len,
                               void* workspace, size_t workspace_bytes, void* stream)
{
    const char* fn = "cache4_attention";
    Cache4Call a;
    int st;
    if ((st = check_type(fn, type, false)) || (st = check_cache(fn, cache, &a.c)) || (st = check_seqs(fn, first, lens, tokens, a.c, &a.s)) ||
        (st = check_heads(fn, a.c, tokens, heads, max_new, max_len)) || (st = check_rows(fn, "q", q, type, tokens, heads, a.c.dim)) ||
        (st = check_rows(fn, "out", out_rows, type, tokens, heads, a.c.dim)) ||
        (st = check_apart(fn, "q", q, heads, out_rows, heads, type, a.c.batch ? tokens : 0, a.c.dim, false)))
        return st;
    if (!std::isfinite(scale)) return fail(TLLM_ERR_SHAPE, "cache4_attention: scale %g", scale);
    a.heads = heads;
    a.scale = scale;
    a.max_new = max_new;
    a.max_len = max_len;
    if (max_len > 0 && max_len < a.s.rows) a.s.rows = max_len;
    a.ws = workspace;
    const size_t need = cache4_workspace(a.c, tokens, heads, max_new, max_len);
    if (need && !workspace) return fail(TLLM_ERR_NULL, "cache4_attention: the workspace is null");
    if (workspace_bytes < need) return fail(TLLM_ERR_SIZE, "cache4_attention: a workspace of %zu bytes, the call needs %zu", workspace_bytes, need);
    if (need && misaligned(workspace, 128)) return fail(TLLM_ERR_ALIGN, "cache4_attention: the workspace must be 128-byte aligned");
    if ((st = check_device()) || (st = error_flag(&a.s))) return st;
    if (type == TLLM_FP16) return launch_cache4_attention<half>(a, in<half>(q), out<half>(out_rows), S(stream));
    return launch_cache4_attention<bf16>(a, in<bf16>(q), out<bf16>(out_rows), S(stream));
}

}  // extern "C"
