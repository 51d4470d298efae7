// Drawing several texts at once from a model (bmb_trainer_generate_batch): prompts in one pass, then a row for each text and step, with
// keys and values in pages of a cache that the texts share.  The reference's generate() (src/train_gpt.cu:46-102) is the same
// for one text; a draw here is its draw.
#include "common.cuh"
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <numeric>
#include <random>
#include <vector>

namespace bmb {
namespace {

// out[row] = wte[token of the row] + wpe[its position]
__global__ void embed_rows_k(float *out, const int *tokens, const int *positions, const float *wte, const float *wpe, long long total, int C) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const long long row = i / C;
    const int c = (int)(i - row * C);
    out[i] = wte[(size_t)tokens[row] * C + c] + wpe[(size_t)positions[row] * C + c];
}

// Slots and positions of tokens that stand one behind the other, as rows of `width` for each request; -1 and 0 behind its last one.
__global__ void spread_rows_k(int *slots_out, int *positions_out, const int *slots, const int *positions, const int *starts, int total, int width) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int request = i / width, at = starts[request] + i % width;
    const bool has = at < starts[request + 1];
    slots_out[i] = has ? slots[at] : -1;
    positions_out[i] = has ? positions[at] : 0;
}

// dst[i] = src[last row of request i's prompt]
__global__ void last_rows_k(float *dst, const float *src, const int *lens, int total, int C, int width) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int request = i / C;
    dst[i] = src[((size_t)request * width + lens[request] - 1) * C + i % C];
}

__global__ void append_k(int *history, int *lens, const int *tokens, const int *grows, int n, int stride) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n && grows[i]) history[(size_t)i * stride + lens[i]++] = tokens[i];
}

// One allocation for the length of a call, handed out in pieces.
struct Arena {
    char *base = nullptr;
    size_t used = 0;
    ~Arena() { if (base) cudaFree(base); }
    template <typename T>
    T *take(size_t count) {
        T *p = reinterpret_cast<T *>((uintptr_t)base + used);
        used += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

constexpr int SV_PAGE = 16;

struct Buffers {
    float *x, *y, *ln, *qkv, *att, *h, *g, *mean, *rstd, *lse, *last, *logits, *probs, *losses;
    int *tokens, *positions, *slots, *packed_slots, *packed_positions, *starts, *lens, *grows, *done, *tables, *stack, *free_pages, *zeros, *history, *history_lens,
        *prompt_lens;
    float *repetition, *frequency, *presence;
    char *k, *v;
    void *workspace;
};

}  // namespace

int generate_texts(const ServeModel &m, int n, const int *host_prompts, int prompt_stride, const int *host_prompt_lens, int steps, unsigned seed,
                   const bmb_batch_sampling &how, int *host_tokens_out) {
    const int C = m.C, NH = m.NH, hs = C / NH, V = m.V, Vp = m.Vp;
    const size_t width = *std::max_element(host_prompt_lens, host_prompt_lens + n), rows = n * width;
    if (rows * 4 * C > 0x7fffffff || (size_t)n * Vp > 0x7fffffff)
        return fail(BMB_E_LIMIT, "trainer_generate_batch: %d prompts of up to %zu tokens are too many at once", n, width);
    const int total = std::accumulate(host_prompt_lens, host_prompt_lens + n, 0);
    size_t pages = 0;
    int longest = 0;
    for (int i = 0; i < n; ++i) {
        pages += (host_prompt_lens[i] + steps + SV_PAGE - 1) / SV_PAGE;
        longest = std::max(longest, host_prompt_lens[i] + steps);
    }
    const int max_pages = (longest + SV_PAGE - 1) / SV_PAGE;
    if (pages * SV_PAGE > 0x7fffffff) return fail(BMB_E_LIMIT, "trainer_generate_batch: %zu pages", pages);
    const size_t element = how.cache_type == BMB_TYPE_FP32 ? 4 : 2, layer_bytes = pages * SV_PAGE * C * element;
    const size_t ws_bytes = bmb_paged_attention_workspace(NH, NH, hs);
    const bool ruled = how.repetition != 1.0f || how.frequency != 0.0f || how.presence != 0.0f;

    Arena arena;
    Buffers b;
    auto lay_out = [&]() {
        b.x = arena.take<float>(rows * C);
        b.y = arena.take<float>(rows * C);
        b.ln = arena.take<float>(rows * C);
        b.att = arena.take<float>(rows * C);
        b.qkv = arena.take<float>(rows * 3 * C);
        b.h = arena.take<float>(rows * 4 * C);
        b.g = arena.take<float>(rows * 4 * C);
        b.mean = arena.take<float>(rows);
        b.rstd = arena.take<float>(rows);
        b.lse = arena.take<float>(rows * NH);
        b.last = arena.take<float>((size_t)n * C);
        b.logits = arena.take<float>((size_t)n * Vp);
        b.probs = arena.take<float>((size_t)n * Vp);
        b.losses = arena.take<float>(n);
        b.tokens = arena.take<int>(rows);
        b.positions = arena.take<int>(rows);
        b.slots = arena.take<int>(rows);
        b.packed_slots = arena.take<int>(total);
        b.packed_positions = arena.take<int>(total);
        b.starts = arena.take<int>(n + 1);
        b.lens = arena.take<int>(n);
        b.grows = arena.take<int>(n);
        b.done = arena.take<int>(n);
        b.tables = arena.take<int>((size_t)n * max_pages);
        b.stack = arena.take<int>(pages);
        b.free_pages = arena.take<int>(1);
        b.zeros = arena.take<int>(n);
        b.history = arena.take<int>((size_t)n * longest);
        b.history_lens = arena.take<int>(n);
        b.prompt_lens = arena.take<int>(n);
        b.repetition = arena.take<float>(n);
        b.frequency = arena.take<float>(n);
        b.presence = arena.take<float>(n);
        b.k = arena.take<char>(layer_bytes * m.L);
        b.v = arena.take<char>(layer_bytes * m.L);
        b.workspace = arena.take<char>(ws_bytes);
    };
    lay_out();                           // (how much it is)
    const size_t bytes = arena.used;
    if (cudaMalloc(&arena.base, bytes) != cudaSuccess) {
        arena.base = nullptr;
        cudaGetLastError();              // (the next launch is not to find it)
        return fail(BMB_E_CUDA, "trainer_generate_batch: no %zu bytes for %d texts of up to %d tokens", bytes, n, longest);
    }
    arena.used = 0;
    lay_out();
    cudaStream_t st = m.st;
    auto upload = [&](void *dst, const void *src, size_t size) -> int {
        BMB_CUDA(cudaMemcpyAsync(dst, src, size, cudaMemcpyHostToDevice, st));      // (nothing that it reads changes before the next synchronise)
        return BMB_OK;
    };
    std::vector<int> tokens(rows, 0), history((size_t)n * longest, 0), ids(pages), ones(n, 1), last(n), ended(n, 0);
    std::vector<float> same(3 * (size_t)n), probs((size_t)n * Vp);
    struct Idle {                        // arena and vectors go when nothing reads or writes them any more
        cudaStream_t st;
        ~Idle() { cudaStreamSynchronize(st); }
    } idle{m.st};
    std::iota(ids.begin(), ids.end(), 0);
    for (int i = 0; i < n; ++i) {
        std::copy_n(host_prompts + (size_t)i * prompt_stride, host_prompt_lens[i], tokens.begin() + i * width);
        std::copy_n(host_prompts + (size_t)i * prompt_stride, host_prompt_lens[i], history.begin() + (size_t)i * longest);
    }
    const int all_pages = (int)pages;
    BMB_TRY(upload(b.tokens, tokens.data(), rows * sizeof(int)));
    BMB_TRY(upload(b.history, history.data(), history.size() * sizeof(int)));
    BMB_TRY(upload(b.history_lens, host_prompt_lens, n * sizeof(int)));
    BMB_TRY(upload(b.prompt_lens, host_prompt_lens, n * sizeof(int)));
    BMB_TRY(upload(b.stack, ids.data(), pages * sizeof(int)));
    BMB_TRY(upload(b.free_pages, &all_pages, sizeof(int)));
    BMB_TRY(upload(b.grows, host_prompt_lens, n * sizeof(int)));
    const float penalties[] = {how.repetition, how.frequency, how.presence};
    float *of_rows[] = {b.repetition, b.frequency, b.presence};
    for (int j = 0; j < 3; ++j) {
        std::fill_n(same.begin() + (size_t)j * n, n, penalties[j]);
        BMB_TRY(upload(of_rows[j], same.data() + (size_t)j * n, n * sizeof(float)));
    }
    BMB_CUDA(cudaMemsetAsync(b.lens, 0, n * sizeof(int), st));
    BMB_CUDA(cudaMemsetAsync(b.zeros, 0, n * sizeof(int), st));
    BMB_CUDA(cudaMemsetAsync(b.tables, 0xff, (size_t)n * max_pages * sizeof(int), st));

    auto product = [&](int M, int N, int K, const float *A, const float *W, const float *bias, float *out) {
        return gemm_any_bias(m.math, m.wflag, 0, 1, 1, M, N, K, 1.0f, A, 0, W, 0, 0.0f, out, 0, bias, st);
    };
    auto cache_of = [&](int l) {
        bmb_kv_cache c{};
        c.k = b.k + l * layer_bytes;
        c.v = b.v + l * layer_bytes;
        c.page_stride = (long long)SV_PAGE * C;
        c.token_stride = C;
        c.head_stride = hs;
        c.type = how.cache_type;
        c.pages = all_pages;
        c.page_size = SV_PAGE;
        c.heads = NH;
        c.head_size = hs;
        return c;
    };
    // The next `columns` tokens of each text (as many of them as `grows` says) through the layers; the last one's row of each in b.last.
    auto forward = [&](int columns, int packed) -> int {
        const int R = n * columns;
        BMB_TRY(bmb_pages_assign(b.tables, b.lens, b.packed_slots, b.packed_positions, nullptr, b.starts, b.free_pages, b.lens, b.grows, b.stack, b.free_pages,
                                 n, max_pages, SV_PAGE, all_pages, packed, st));
        BMB_TRY(launch(false, spread_rows_k, ceil_div(R, 256), 256, 0, st, b.slots, b.positions, b.packed_slots, b.packed_positions, b.starts, R, columns));
        BMB_TRY(launch(false, embed_rows_k, ceil_div((long long)R * C, 256), 256, 0, st, b.x, b.tokens, b.positions, m.wte, m.wpe, (long long)R * C, C));
        float *x = b.x, *y = b.y;
        BMB_TRY(bmb_layernorm_forward(b.ln, b.mean, b.rstd, x, m.ln1w, m.ln1b, R, C));
        for (int l = 0; l < m.L; ++l) {
            const size_t c1 = (size_t)l * C, w = c1 * C;
            BMB_TRY(product(R, 3 * C, C, b.ln, m.qkvw + 3 * w, m.qkvb + 3 * c1, b.qkv));
            const bmb_kv_cache cache = cache_of(l);
            BMB_TRY(bmb_paged_kv_write(&cache, b.qkv + C, b.qkv + 2 * C, 3 * C, b.slots, R, st));
            if (columns > 1)             // a prompt's rows see one another; rows behind its end see it, and nobody sees them
                BMB_TRY(flash_forward(m.attention, 0, b.att, b.lse, b.qkv, n, columns, C, NH, false));
            else
                BMB_TRY(bmb_paged_attention(b.att, nullptr, b.qkv, &cache, b.tables, b.lens, n, NH, 3 * C, C, max_pages, 1.0f / sqrtf((float)hs), b.workspace,
                                            ws_bytes, st));
            BMB_TRY(product(R, C, C, b.att, m.apw + w, m.apb + c1, b.h));
            BMB_TRY(bmb_residual_layernorm_forward(y, b.ln, b.mean, b.rstd, x, b.h, m.ln2w + c1, m.ln2b + c1, R, C));
            BMB_TRY(product(R, 4 * C, C, b.ln, m.fcw + 4 * w, m.fcb + 4 * c1, b.h));
            BMB_TRY(bmb_gelu_forward(b.g, b.h, 4 * R * C));
            BMB_TRY(product(R, C, 4 * C, b.g, m.fpw + 4 * w, m.fpb + c1, b.h));
            const bool end = l + 1 == m.L;
            BMB_TRY(bmb_residual_layernorm_forward(x, b.ln, b.mean, b.rstd, y, b.h, end ? m.lnfw : m.ln1w + c1 + C, end ? m.lnfb : m.ln1b + c1 + C, R, C));
        }
        if (columns > 1)
            BMB_TRY(launch(false, last_rows_k, ceil_div((long long)n * C, 256), 256, 0, st, b.last, b.ln, b.prompt_lens, n * C, C, columns));
        return product(n, Vp, C, columns > 1 ? b.last : b.ln, m.wte_w, nullptr, b.logits);
    };

    std::vector<std::mt19937> rng;
    for (int i = 0; i < n; ++i) rng.emplace_back(seed + i);
    std::uniform_real_distribution<float> uni(0.0f, 1.0f);
    std::fill(host_tokens_out, host_tokens_out + (size_t)n * steps, -1);
    int left = n;
    for (int s = 0; s < steps && left > 0; ++s) {
        BMB_TRY(s == 0 ? forward((int)width, total) : forward(1, n));
        if (ruled) {
            bmb_logit_rules r{};
            r.history = b.history;
            r.history_lens = b.history_lens;
            r.prompt_lens = b.prompt_lens;
            r.repetition = b.repetition;
            r.frequency = b.frequency;
            r.presence = b.presence;
            r.history_stride = longest;
            BMB_TRY(bmb_logits_adjust(b.logits, b.logits, n, V, Vp, &r, st));
        }
        BMB_TRY(bmb_softmax_crossentropy_forward(b.probs, b.losses, b.logits, b.zeros, n, V, Vp));
        BMB_CUDA(cudaMemcpyAsync(probs.data(), b.probs, probs.size() * sizeof(float), cudaMemcpyDeviceToHost, st));
        BMB_CUDA(cudaStreamSynchronize(st));
        std::fill(ended.begin(), ended.end(), 0);
        int ending = 0;
        for (int i = 0; i < n; ++i) {
            if (!ones[i]) continue;
            last[i] = draw_token(&probs[(size_t)i * Vp], V, how.temperature, uni(rng[i]));
            host_tokens_out[(size_t)i * steps + s] = last[i];
            if (last[i] == how.stop_token) {
                ones[i] = 0;
                ended[i] = 1;
                ++ending;
                --left;
            }
        }
        if (s + 1 == steps) break;
        BMB_TRY(upload(b.tokens, last.data(), n * sizeof(int)));
        BMB_TRY(upload(b.grows, ones.data(), n * sizeof(int)));
        if (ending) {
            BMB_TRY(upload(b.done, ended.data(), n * sizeof(int)));
            BMB_TRY(bmb_pages_release(b.stack, b.free_pages, b.lens, b.free_pages, b.lens, b.tables, b.done, n, max_pages, SV_PAGE, all_pages, st));
        }
        if (ruled) BMB_TRY(launch(false, append_k, ceil_div(n, 256), 256, 0, st, b.history, b.history_lens, b.tokens, b.grows, n, longest));
    }
    return BMB_OK;
}

int draw_token(float *probs, int V, float temperature, float coin) {
    if (temperature != 1.0f) {
        // Cold draws: where even the largest power is below fp32's normal numbers (0.1^100), the powers are those of shares of the largest.
        const float top = *std::max_element(probs, probs + V);
        const float unit = top > 0.0f && powf(top, 1.0f / temperature) < FLT_MIN ? top : 1.0f;
        float sum = 0.0f;
        for (int i = 0; i < V; ++i) { probs[i] = powf(probs[i] / unit, 1.0f / temperature); sum += probs[i]; }
        for (int i = 0; i < V; ++i) probs[i] /= sum;
    }
    float cdf = 0.0f;
    for (int i = 0; i < V; ++i) { cdf += probs[i]; if (coin < cdf) return i; }
    return V - 1;
}

}  // namespace bmb
