// draft.hip - steps with drafted tokens: the trees' masks and positions, the drafts' verification, and moving the accepted rows
// together in the caches (include/gcq_draft.h; append and attention of such rows are paged.hip's and paged_attn.hip's).
#include <algorithm>

#include "paged.h"

#include "../../include/gcq_draft.h"

namespace gcq {

namespace {

constexpr int kMaxRows = GCQ_DRAFT_MAX_ROWS;

// The rows of sequence s, no more than max_rows; none where starts do not ascend.
struct Rows {
    int r0, n;
};
__device__ __forceinline__ Rows rows_of(const int32_t * starts, int s, int n_rows, int max_rows) {
    const int r0 = starts[s], r1 = min(starts[s + 1], n_rows);
    return {r0, r0 < 0 || r1 <= r0 ? 0 : min(r1 - r0, max_rows)};
}

// ------------------------------------------------------------------------------------ trees

struct TreeArgs {
    const int32_t * starts, * past, * parents;
    int n_rows, max_rows, window, ld;
    int32_t * positions;
    uint32_t * mask;
};

// A workgroup to a sequence. A row's ancestors by doubling: with those up to 2^k levels above known, and the row there, another round
// takes in that row's; log2 of the deepest row's depth rounds, whatever the order of the rows. Masks eight words at a time, so that
// 1024 rows fit. Latency: a few rounds in LDS.
__global__ __launch_bounds__(256) void k_draft_tree(const TreeArgs a) {
    constexpr int W = 8, T = 256, N = kMaxRows / T;  // words at a time, threads, rows of a thread
    __shared__ uint32_t seen[kMaxRows][W + 1];
    __shared__ int16_t up[kMaxRows];
    __shared__ int16_t depth[kMaxRows];
    const int s = blockIdx.x, tid = threadIdx.x;
    const Rows w = rows_of(a.starts, s, a.n_rows, a.max_rows);
    if (w.n == 0) return;
    for (int w0 = 0; w0 < a.ld; w0 += W) {
        for (int j = tid; j < w.n; j += T) {
            const int parent = a.parents[w.r0 + j];
            up[j] = parent >= 0 && parent < j ? parent : -1;
            if (w0 == 0) depth[j] = parent >= 0 && parent < j;  // rows above it, as far as they are known
#pragma unroll
            for (int x = 0; x < W; x++) seen[j][x] = j / 32 == w0 + x ? 1u << (j % 32) : 0;
        }
        __syncthreads();
        for (;;) {
            int above[N], further[N], more[N];
            uint32_t bits[N][W];
            bool any = false;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int j = tid + T * n;
                above[n] = j < w.n ? up[j] : -1;
                if (above[n] < 0) continue;
                any = true;
                further[n] = up[above[n]];
                more[n] = depth[above[n]];
#pragma unroll
                for (int x = 0; x < W; x++) bits[n][x] = seen[above[n]][x];
            }
            if (!__syncthreads_or(any)) break;
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int j = tid + T * n;
                if (above[n] < 0) continue;
                up[j] = further[n];
                if (w0 == 0) depth[j] += more[n];
#pragma unroll
                for (int x = 0; x < W; x++) seen[j][x] |= bits[n][x];
            }
            __syncthreads();
        }
        for (int i = tid; i < w.n * W; i += T) {
            const int j = i / W, x = i % W;
            if (w0 + x >= a.ld) continue;
            uint32_t m = seen[j][x];
            if (a.window && depth[j] >= a.window)
                for (uint32_t left = m; left; left &= left - 1) {
                    const int b = __builtin_ctz(left);
                    if (depth[j] - depth[32 * (w0 + x) + b] >= a.window) m &= ~(1u << b);
                }
            a.mask[(int64_t) (w.r0 + j) * a.ld + w0 + x] = m;
        }
        if (w0 == 0)
            for (int j = tid; j < w.n; j += T) a.positions[w.r0 + j] = (int) min((int64_t) a.past[s] + depth[j], (int64_t) INT32_MAX);
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------- verification

struct VerifyArgs {
    const int32_t * starts, * parents, * tokens;
    const float * logits, * draft, * temperature, * coins;
    int64_t ld, draft_ld;
    int n_rows, V, max_rows, max_path;
    int32_t * count, * rows, * out;
};

// A logit as it counts: NaN as -inf, +inf as the largest float.
__device__ __forceinline__ float logit(float x) { return x == x ? fminf(x, 3.402823466e38f) : -INFINITY; }

// A row's softmax: its largest logit, the lowest that has it, 1 / temperature, and the sum of exp((l - m) inv).
struct Soft {
    float m;
    int top;
    double inv, sum;
    __device__ __forceinline__ double weight(float x) const {
        const float l = logit(x);
        return l == -INFINITY ? 0.0 : exp(((double) l - (double) m) * inv);
    }
    __device__ __forceinline__ double p(float x) const { return sum > 0.0 ? weight(x) / sum : 0.0; }
};

constexpr int kT = 1024, kWaves = kT / 64;

__device__ __forceinline__ double block_sum(double v, double * red) {
    v = wave_sum_d(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kWaves; w++) s += red[w];
    __syncthreads();
    return s;
}

__device__ __forceinline__ Soft soft_of(const float * x, int V, double inv, bool sums, double * red) {
    float * rm = (float *) red;
    int * ri = (int *) red + kWaves;
    Soft z{-INFINITY, 0x7fffffff, inv, 0.0};
    for (int i = threadIdx.x; i < V; i += kT) argmax_take(z.m, z.top, logit(x[i]), i);
    for (int o = 32; o > 0; o >>= 1) argmax_take(z.m, z.top, __shfl_xor(z.m, o, 64), __shfl_xor(z.top, o, 64));
    if ((threadIdx.x & 63) == 0) rm[threadIdx.x >> 6] = z.m, ri[threadIdx.x >> 6] = z.top;
    __syncthreads();
    for (int w = 0; w < kWaves; w++) argmax_take(z.m, z.top, rm[w], ri[w]);
    __syncthreads();
    if (!sums || z.m == -INFINITY) return z;
    double s = 0.0;
    for (int i = threadIdx.x; i < V; i += kT) s += z.weight(x[i]);
    z.sum = block_sum(s, red);
    return z;
}

// A workgroup walks a sequence's tree, all of a row's logits at a time.
//   r after k fallen drafts is w_k / c_k, w_k = max(p - C_k q, 0), c_k its sum, C_0 = 0 and C_k+1 = C_k + c_k, since
//   max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0; for guesses that were not drawn p without those tokens.
__global__ __launch_bounds__(kT) void k_draft_verify(const VerifyArgs a) {
    __shared__ double red[kWaves];
    __shared__ int fallen[kMaxRows];  // their tokens
    __shared__ int child;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Rows w = rows_of(a.starts, s, a.n_rows, a.max_rows);
    const float t = a.temperature ? a.temperature[s] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const double inv = greedy ? 1.0 : 1.0 / (double) t;
    int n = 0;
    for (int u = 0; w.n && n < a.max_path;) {
        const float * x = a.logits + (int64_t) (w.r0 + u) * a.ld;
        const float * y = a.draft ? a.draft + (int64_t) (w.r0 + u) * a.draft_ld : nullptr;
        const Soft p = soft_of(x, a.V, inv, !greedy, red);
        Soft q{};
        bool have_q = false;
        double C = 0.0, c = 1.0;
        int gone = 0, taken = -1;
        const auto left = [&](int i) {  // w_k
            if (!y) {
                for (int f = 0; f < gone; f++)
                    if (fallen[f] == i) return 0.0;
                return p.p(x[i]);
            }
            return C == 0.0 ? p.p(x[i]) : fmax(p.p(x[i]) - C * q.p(y[i]), 0.0);
        };
        for (int c0 = u;;) {  // the children in order
            if (tid == 0) child = w.n;
            __syncthreads();
            for (int j = c0 + 1 + tid; j < w.n; j += kT)
                if (a.parents[w.r0 + j] == u) {
                    atomicMin(&child, j);
                    break;
                }
            __syncthreads();
            c0 = child;
            __syncthreads();
            if (c0 >= w.n) break;
            const int token = a.tokens[w.r0 + c0];
            const bool known = token >= 0 && token < a.V;
            if (greedy) {
                if (p.m > -INFINITY && token == p.top) taken = c0;
            } else if (known) {
                if (y && !have_q) q = soft_of(y, a.V, inv, true, red), have_q = true;
                if ((double) a.coins[w.r0 + c0] * c * (y ? q.p(y[token]) : 1.0) < left(token)) taken = c0;
            }
            if (taken >= 0) break;
            if (greedy || (!y && !known)) continue;
            if (y) {
                if (!have_q) q = soft_of(y, a.V, inv, true, red), have_q = true;
                C += c;
            } else if (tid == 0) fallen[gone] = token;
            if (!y) gone++;
            __syncthreads();
            double sum = 0.0;
            for (int i = tid; i < a.V; i += kT) sum += left(i);
            c = block_sum(sum, red);
        }
        int next = -1;
        if (taken >= 0) next = a.tokens[w.r0 + taken];
        else if (p.m > -INFINITY) {
            if (greedy) next = p.top;
            else {
                if (!(c > 0.0)) C = 0.0, gone = 0;
                // a wavefront's run of tokens; then the run that holds the sum in question
                const int run = (a.V + kWaves - 1) / kWaves, i0 = min(wave * run, a.V), i1 = min(i0 + run, a.V);
                double sum = 0.0;
                for (int i = i0 + lane; i < i1; i += 64) sum += left(i);
                sum = wave_sum_d(sum);
                if (lane == 0) red[wave] = sum;
                if (tid == 0) child = -1;
                __syncthreads();
                double total = 0.0, below = 0.0;
                for (int v = 0; v < kWaves; v++) total += red[v];
                const float coin = a.coins[w.r0];
                const double at = (coin > 0.0f ? fmin((double) coin, 1.0 - 0x1p-24) : 0.0) * total;
                int mine = -1;
                for (int v = 0; v < kWaves; v++) {
                    if (red[v] > 0.0) {
                        mine = v;
                        if (below + red[v] > at) break;
                    }
                    below += red[v];
                }
                if (mine == wave) {
                    if (!(below + red[mine] > at)) below -= red[mine];
                    int last = -1;
                    for (int i = i0; i < i1; i += 64) {
                        double v = i + lane < i1 ? left(i + lane) : 0.0, sums = v;
                        for (int o = 1; o < 64; o <<= 1) {
                            const double b = __shfl_up(sums, o, 64);
                            if (lane >= o) sums += b;
                        }
                        const uint64_t hit = __ballot(v > 0.0 && below + sums > at), some = __ballot(v > 0.0);
                        if (some) last = i + 63 - __builtin_clzll(some);
                        if (hit) {
                            last = i + __builtin_ctzll(hit);
                            break;
                        }
                        below += __shfl(sums, 63, 64);
                    }
                    if (lane == 0) child = last;
                }
                __syncthreads();
                next = child;
                __syncthreads();
            }
        }
        if (tid == 0) {
            a.rows[(int64_t) s * a.max_path + n] = u;
            a.out[(int64_t) s * a.max_path + n] = next;
        }
        n++;
        if (taken < 0) break;
        u = taken;
    }
    if (tid == 0) a.count[s] = n;
    for (int i = n + tid; i < a.max_path; i += kT) a.rows[(int64_t) s * a.max_path + i] = a.out[(int64_t) s * a.max_path + i] = -1;
}

// ------------------------------------------------------------------------------------ move

constexpr int kCaches = 64;  // of a launch

struct MoveArgs {
    Paged p;
    uint8_t * data[kCaches];
    const int32_t * count, * rows;
    int64_t ld;
    int max_keep;
};

// A wavefront moves one sequence's tokens of one KV head in one cache: a lane has the same code bytes of every token. In order of the
// targets, so that nothing is written before it is read: an entry's source is not below its own number, so no earlier target.
template <int D>
__global__ __launch_bounds__(64) void k_paged_move(const MoveArgs a) {
    constexpr int B = D / 64 > 0 ? D / 64 : 1;
    const int lane = threadIdx.x, s = blockIdx.x / a.p.Hkv, hk = blockIdx.x % a.p.Hkv;
    Paged p = a.p;
    p.data = a.data[blockIdx.y];
    const int n = min(a.count[s], a.max_keep);
    const int64_t past = a.p.past[s];
    for (int i = 0; i < n; i++) {
        const int j = a.rows[s * a.ld + i];
        if (j <= i) continue;
        const int64_t src = paged_tile(p, s, past + j, hk, D), dst = paged_tile(p, s, past + i, hk, D);
        if (src < 0 || dst < 0) continue;
        const int ts = (int) (past + j) & 31, td = (int) (past + i) & 31;
#pragma unroll
        for (int b = 0; b < B; b++) {
            const int e = lane + 64 * b;
            if (e < D / 2) {
                p.data[dst + paged_k_byte<D>(td, e)] = p.data[src + paged_k_byte<D>(ts, e)];
                p.data[dst + paged_v_byte<D>(td, e)] = p.data[src + paged_v_byte<D>(ts, e)];
            }
        }
        if (lane < D / 16) {  // scales: of K, then of V, whose lie as if they were further blocks
            const uint16_t d = *reinterpret_cast<const uint16_t *>(p.data + src + paged_k_scale<D>(ts, lane));
            *reinterpret_cast<uint16_t *>(p.data + dst + paged_k_scale<D>(td, lane)) = d;
        }
    }
}

template <class F>
void with_head_dim(int D, F && f) {
    if (D == 64) f(std::integral_constant<int, 64>{});
    else if (D == 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 256>{});
}

size_t verify_workspace(int n_seq, int64_t n_rows, int64_t V, int64_t max_rows) {
    paged_require(n_seq > 0 && n_seq < (1 << 30), "draft_verify: at least one sequence");
    paged_require(n_rows >= 0 && n_rows < (1 << 30), "draft_verify: n_rows out of range");
    paged_require(V > 0 && V < (1 << 30), "draft_verify: n_vocab out of range");
    paged_require(max_rows > 0 && std::min(max_rows, n_rows) <= kMaxRows, "draft_verify: max_rows must be 1 .. 1024");
    return 256;
}

}  // namespace

}  // namespace gcq

using namespace gcq;

extern "C" {

int gcq_draft_tree(const gcq_paged_batch * batch, int64_t n_rows, const int32_t * parents, int64_t max_rows, int window,
                   int32_t * positions, uint32_t * mask, int64_t ld_mask, void * stream) {
    return guarded([&] {
        paged_need(batch, "batch");
        paged_require(batch->n_seq > 0, "draft_tree: at least one sequence");
        paged_require(n_rows >= 0 && n_rows < (1 << 30), "draft_tree: n_rows out of range");
        paged_require(max_rows > 0, "draft_tree: max_rows must be positive");
        paged_require(ld_mask > 0 && ld_mask <= kMaxRows / 32, "draft_tree: ld_mask must be 1 .. 32");
        paged_require(std::min(max_rows, n_rows) <= 32 * ld_mask, "draft_tree: max_rows past the mask's bits");
        paged_require(window >= 0, "draft_tree: window must not be negative");
        if (n_rows == 0) return;
        paged_need(batch->starts, "starts", 4);
        paged_need(batch->past, "past", 4);
        paged_need(parents, "parents", 4);
        paged_need(positions, "positions", 4);
        paged_need(mask, "mask", 4);
        const TreeArgs a{batch->starts, batch->past, parents, (int) n_rows, (int) std::min(max_rows, n_rows), window, (int) ld_mask,
                         positions, mask};
        k_draft_tree<<<paged_grid(batch->n_seq, 256), 256, 0, as_stream(stream)>>>(a);
        check_launch("draft tree");
    });
}

size_t gcq_draft_verify_workspace(int n_seq, int64_t n_rows, int64_t n_vocab, int64_t max_rows) {
    size_t n = 0;
    guarded([&] { n = verify_workspace(n_seq, n_rows, n_vocab, max_rows); });
    return n;
}

int gcq_draft_verify(const int32_t * starts, int n_seq, int64_t n_rows, const int32_t * parents, const int32_t * tokens,
                     const float * logits, int64_t ld, const float * draft_logits, int64_t draft_ld, int64_t n_vocab,
                     const float * temperature, const float * coins, int64_t max_rows, int max_path, int32_t * count,
                     int32_t * rows, int32_t * tokens_out, void * ws, size_t ws_size, void * stream) {
    return guarded([&] {
        const size_t need_ws = verify_workspace(n_seq, n_rows, n_vocab, max_rows);
        paged_require(max_path > 0, "draft_verify: max_path must be positive");
        paged_need(starts, "starts", 4);
        paged_need(count, "count", 4);
        paged_need(rows, "rows", 4);
        paged_need(tokens_out, "tokens_out", 4);
        if (n_rows) {
            paged_need(parents, "parents", 4);
            paged_need(tokens, "tokens", 4);
            paged_need(logits, "logits", 4);
            paged_need(coins, "coins", 4);
            paged_require(ld >= n_vocab, "draft_verify: rows of logits overlap");
            if (draft_logits) {
                paged_need(draft_logits, "draft_logits", 4);
                paged_require(draft_ld >= n_vocab, "draft_verify: rows of draft_logits overlap");
            }
            if (temperature) paged_need(temperature, "temperature", 4);
        }
        paged_need(ws, "workspace", 256);
        if (ws_size < need_ws) fail("workspace of " + std::to_string(ws_size) + " bytes, need " + std::to_string(need_ws));
        VerifyArgs a{};
        a.starts = starts, a.parents = parents, a.tokens = tokens, a.logits = logits, a.ld = ld, a.draft = draft_logits, a.draft_ld = draft_ld;
        a.temperature = temperature, a.coins = coins, a.n_rows = (int) n_rows, a.V = (int) n_vocab;
        a.max_rows = (int) std::min<int64_t>(max_rows, std::max<int64_t>(n_rows, 1)), a.max_path = max_path;
        a.count = count, a.rows = rows, a.out = tokens_out;
        k_draft_verify<<<paged_grid(n_seq, kT), kT, 0, as_stream(stream)>>>(a);
        check_launch("draft verify");
    });
}

int gcq_paged_move(const gcq_paged_cache * const * caches, int n_caches, const gcq_paged_batch * batch, const int32_t * count,
                   const int32_t * rows, int64_t ld_rows, int max_keep, void * stream) {
    return guarded([&] {
        paged_need(caches, "caches");
        paged_require(n_caches > 0, "paged_move: at least one cache");
        paged_need(count, "count", 4);
        paged_need(rows, "rows", 4);
        paged_require(max_keep >= 0 && ld_rows >= max_keep, "paged_move: ld_rows >= max_keep >= 0");
        for (int c0 = 0; c0 < n_caches; c0++) {
            const Paged p = paged_view(caches[c0], batch, 1);
            (void) p;
            paged_require(caches[c0]->n_pages == caches[0]->n_pages && caches[c0]->page_size == caches[0]->page_size &&
                              caches[c0]->n_head_kv == caches[0]->n_head_kv && caches[c0]->head_dim == caches[0]->head_dim,
                          "paged_move: the caches must be of one shape");
        }
        if (max_keep == 0) return;
        MoveArgs a{};
        a.p = paged_view(caches[0], batch, 1);
        a.count = count, a.rows = rows, a.ld = ld_rows, a.max_keep = max_keep;
        for (int c0 = 0; c0 < n_caches; c0 += kCaches) {
            const int n = std::min(n_caches - c0, kCaches);
            for (int i = 0; i < n; i++) a.data[i] = (uint8_t *) caches[c0 + i]->data;
            const unsigned x = paged_grid((int64_t) batch->n_seq * a.p.Hkv * n, 64) / n;
            with_head_dim(caches[0]->head_dim, [&](auto d) { k_paged_move<decltype(d)::value><<<dim3(x, n), 64, 0, as_stream(stream)>>>(a); });
            check_launch("paged move");
        }
    });
}

}  // extern "C"
