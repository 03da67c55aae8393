// draft.hip - steps with drafted tokens: the trees' masks and positions, the drafts' verification, and moving the accepted rows
// together in the caches (include/gcq_draft.h; append and attention of such rows are paged.hip's and paged_attn.hip's).
#include <algorithm>
#include <cmath>

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
//
// Three launches. k_verify_begin puts the rows in order, the sequences' first rows first, then their second ones, .. k_verify_rows
// takes each row's logits in parts, a workgroup to a part: the largest and the sum of exponentials, of the target's and, where a
// row has children, the drafter's. Whichever of a row's workgroups ends last has the row's softmax and decides which child stands,
// which depends on nothing but the row. Rows that an earlier decision has cut off from the path are passed over if it is
// known by then: in this order, where rows are many, it mostly is (nobody waits for it, and no result depends on it).
// k_verify_walk, some workgroups to a sequence, follows the decisions from the root on and draws the last row's token.
//
// r after k fallen drafts is w_k / c_k, w_k = max(p - C_k q, 0), c_k its sum, C_0 = 0 and C_k+1 = C_k + c_k, since
// max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0: one sum over the vocabulary for each that falls, which the walk makes
// for the rows on the path alone.
//
// In 64 bits: a token's border in the cumulative sum would be off by 2^-25 or so in 32, and 10^5 borders then put a drawn token wrong
// once in some hundred draws.

constexpr int kT = 256;
constexpr int kDraw = 16;  // values of a thread in the walk

// What became of a row: the child that stands (>= 0), or
enum : int { kNone = -1, kOpen = -2, kCut = -3, kFell = -16 };  // kFell - j: child j fell, others are left, r's sum is not known

struct __align__(64) RowState {
    double sum_p, sum_q, C;  // sums of exp((l - m) / t)
    float m_p, m_q;
    int top, next, arrived;
};
struct __align__(16) PartSums {
    double p, q;
    float m_p, m_q;
    int top, pad;
};
constexpr int kPartWords = sizeof(PartSums) / 8;
struct SeqState {
    int arrived, done;
};
struct __align__(16) Item {  // a row in its order
    int r, s, j, parent;  // parent < 0: none
    int r0, n;            // its sequence's rows
    float t;              // temperature
    int child;            // the first; n: none
};
struct __align__(16) Drawn {
    double w, p;
};
constexpr int kDrawnWords = sizeof(Drawn) / 8;

struct VerifyArgs {
    const int32_t * starts, * parents, * tokens;
    const float * logits, * draft, * temperature, * coins;
    int64_t ld, draft_ld;
    int n_seq, n_rows, V, max_rows, max_path, parts, draws;
    bool vec, last;  // rows of whole 16-byte pieces; the last walk
    int32_t * count, * rows, * out;
    int * n_items;
    Item * items;
    RowState * state;
    PartSums * sums;
    SeqState * seq;
    Drawn * drawn;
    double roots[16];  // 2^(i / 16)
};

// exp by a sixteenth of a power of two from LDS (a bank of its own each) and five terms of exp's series on what is left: |z| <= ln 2 / 32, the
// sixth is 2^-43. 12 operations of 64 bits; the library's takes about twice as many.
struct Soft {
    const double * roots;  // LDS
    double scale, m, inv;  // 16 / (t ln 2), the row's largest logit, 1 / its sum
    bool huge;             // some logit is infinite
    __device__ __forceinline__ double weight(float l) const {
        if (huge) l = fminf(l, 3.402823466e38f);
        const double x = ((double) l - m) * scale, t = x + 0x1.8p52, r = x - (t - 0x1.8p52);
        const int n = (int) (uint32_t) __double_as_longlong(t);
        constexpr double k = 0.043321698784996581;  // ln 2 / 16
        double y = fma(r, k * k * k * k * k / 120, k * k * k * k / 24);
        y = fma(r, y, k * k * k / 6);
        y = fma(r, y, k * k / 2);
        y = fma(r, y, k);
        y = fma(r, y, 1.0) * roots[n & 15];
        y = __hiloint2double(__double2hiint(y) + ((n >> 4) << 20), __double2loint(y));
        return x > -16000.0 ? y : 0.0;  // (nor for -inf and NaN)
    }
    __device__ __forceinline__ double p(float l) const { return weight(l) * inv; }
};
__device__ __forceinline__ Soft soft(const double * roots, double inv_t, float m, double sum) {
    return {roots, inv_t * 23.083120654223414, (double) m, sum > 0.0 ? 1.0 / sum : 0.0, m >= 3.402823466e38f};
}

// N values x[i ..), those at V and beyond -inf.
template <int N>
__device__ __forceinline__ void values(const float * x, int i, int V, bool vec, float (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        if (vec && i + e + 3 < V) *reinterpret_cast<float4 *>(v + e) = *reinterpret_cast<const float4 *>(x + i + e);
        else
#pragma unroll
            for (int c = 0; c < 4; c++) v[e + c] = i + e + c < V ? x[i + e + c] : -INFINITY;
    }
}

template <class T>
__device__ __forceinline__ T agent_load(const T * p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T>
__device__ __forceinline__ void agent_store(T * p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// What workgroups tell each other within a launch goes past the XCDs' L2s, word by word: a fence would write back and drop a whole L2, some
// 40 ns each and one after the other (5120 workgroups 220 us; so 60).
template <class T>
__device__ __forceinline__ void share(T * to, const T & v) {
    static_assert(sizeof(T) % 8 == 0, "words of 8 bytes");
    uint64_t w[sizeof(T) / 8];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 8; i++) agent_store(reinterpret_cast<uint64_t *>(to) + i, w[i]);
}
template <class T>
__device__ __forceinline__ T shared(const T * from) {
    uint64_t w[sizeof(T) / 8];
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 8; i++) w[i] = agent_load(reinterpret_cast<const uint64_t *>(from) + i);
    T v;
    __builtin_memcpy(&v, w, sizeof(T));
    return v;
}
// Whether this workgroup is the last of n to arrive, after thread 0 has shared what it has (all threads together). The stores have reached
// memory before the count is raised; who reads the last count reads them there.
__device__ __forceinline__ bool last_of(int * arrived, int n, int * flag) {
    if (threadIdx.x == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        *flag = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
    }
    __syncthreads();
    return *flag;
}

// The first child of row u after row `from` of sequence w, w.n if there is none (a whole wavefront).
__device__ __forceinline__ int child_after(const int32_t * parents, const Rows & w, int u, int from) {
    const int lane = threadIdx.x & 63;
    for (int j0 = from + 1; j0 < w.n; j0 += 64) {
        const uint64_t at = __ballot(j0 + lane < w.n && parents[w.r0 + min(j0 + lane, w.n - 1)] == u);
        if (at) return j0 + __builtin_ctzll(at);
    }
    return w.n;
}

// A wavefront to a row: its place in the order, and its state.
__global__ __launch_bounds__(kT) void k_verify_begin(const VerifyArgs a) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * (kT / 64) + (threadIdx.x >> 6);
    for (int s = blockIdx.x * kT + threadIdx.x; s < a.n_seq; s += gridDim.x * kT) a.seq[s] = SeqState{};
    if (r >= a.n_rows) return;
    if (lane == 0) a.state[r] = {0.0, 0.0, 0.0, -INFINITY, -INFINITY, 0x7fffffff, kOpen, 0};
    const auto load = [&](int s0) { return s0 + lane < a.n_seq ? rows_of(a.starts, s0 + lane, a.n_rows, a.max_rows) : Rows{}; };
    const Rows first = load(0);
    Rows w{}, x = first;
    int s = -1, before = 0, all = 0;
    for (int s0 = 0; s0 < a.n_seq && s < 0; s0 += 64) {
        if (s0) x = load(s0);
        const uint64_t at = __ballot(r >= x.r0 && r < x.r0 + x.n);
        if (!at) continue;
        const int l = __builtin_ctzll(at);
        s = s0 + l;
        w = {__builtin_amdgcn_readlane(x.r0, l), __builtin_amdgcn_readlane(x.n, l)};
    }
    if (s < 0 && r > 0) return;
    const int j = r - w.r0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64) {
        const int n = s0 ? load(s0).n : first.n;
        before += min(n, j) + (n > j && s0 + lane < s);
        all += n;
    }
    before = wave_isum(before);
    if (r == 0) {
        all = wave_isum(all);
        if (lane == 0) *a.n_items = all;
    }
    if (s < 0 || before >= a.n_rows) return;
    const int parent = a.parents[r], child = child_after(a.parents, w, j, j);
    // (rows but the first that follow nothing: no path leads there)
    if (lane == 0) a.items[before] = {r, s, j, parent >= 0 && parent < j ? parent : -1, w.r0, w.n, a.temperature ? a.temperature[s] : 1.0f, child};
}

// A row's children as lanes have them: of the 64 rows from j0 on, which are the row's, their tokens, coins and logits (a wavefront).
struct Children {
    uint64_t at;
    int token;
    float coin, x, y;  // the target's logit, the drafter's
};
__device__ __forceinline__ Children children(const VerifyArgs & a, const Rows & w, int u, int j0) {
    const int lane = threadIdx.x & 63, j = min(j0 + lane, w.n - 1);
    Children c{0, -1, 0.0f, -INFINITY, -INFINITY};
    const bool mine = j0 + lane < w.n && a.parents[w.r0 + j] == u;
    c.at = __ballot(mine);
    if (mine) {
        c.token = a.tokens[w.r0 + j];
        c.coin = a.coins[w.r0 + j];
        if (c.token >= 0 && c.token < a.V) {
            c.x = a.logits[(w.r0 + u) * a.ld + c.token];
            if (a.draft) c.y = a.draft[(w.r0 + u) * a.draft_ld + c.token];
        }
    }
    return c;
}
// The next child of a drawn row, row `from` having fallen last and r's sum c being known; k: the children from row j0 on.
__device__ __forceinline__ void decide_drawn(const VerifyArgs & a, const Rows & w, int u, int from, double c, const Soft & p, const Soft & q,
                                             Children k, int j0, RowState & z) {
    z.next = kNone;
    for (; j0 < w.n; k = children(a, w, u, j0 += 64)) {
        const uint64_t left = from < j0 ? k.at : from - j0 >= 63 ? 0 : k.at >> (from - j0 + 1) << (from - j0 + 1);
        if (!left) {
            if (j0 + 64 >= w.n) return;
            continue;
        }
        const int l = __builtin_ctzll(left), token = __builtin_amdgcn_readlane(k.token, l);
        const double pt = p.p(readlane_f(k.x, l)), qt = q.p(readlane_f(k.y, l));
        if (token >= 0 && token < a.V && (double) readlane_f(k.coin, l) * c * qt < fmax(pt - z.C * qt, 0.0)) {
            z.next = j0 + l;
            return;
        }
        z.C += c;
        if (left & (left - 1) || child_after(a.parents, w, u, j0 + 63) < w.n) z.next = kFell - (j0 + l);
        return;
    }
}
// All children of a row whose drafts were not drawn.
__device__ __forceinline__ int decide_guessed(const VerifyArgs & a, const Rows & w, int u, const Soft & p, Children k) {
    const int lane = threadIdx.x & 63;
    double left = 1.0;  // what the fallen leave
    for (int j0 = u + 1; j0 < w.n;) {
        const double pt = p.p(k.x);
        for (uint64_t at = k.at; at; at &= at - 1) {
            const int l = __builtin_ctzll(at), t = __builtin_amdgcn_readlane(k.token, l);
            double v = readlane_d(pt, l);
            bool before = (k.at >> lane & 1) && lane < l && k.token == t;  // (fell already)
            for (int i = u + 1 + lane; i < j0; i += 64) before = before || (a.parents[w.r0 + i] == u && a.tokens[w.r0 + i] == t);
            if (__any(before)) v = 0.0;
            if ((double) readlane_f(k.coin, l) * left < v) return j0 + l;
            left -= v;
        }
        if ((j0 += 64) < w.n) k = children(a, w, u, j0);
    }
    return kNone;
}

template <int NV>
__global__ __launch_bounds__(kT) void k_verify_rows(const VerifyArgs a) {
    __shared__ double roots[16], red[2][kT / 64];
    __shared__ float redm[2][kT / 64];
    __shared__ int redt[kT / 64], flag;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = blockIdx.x % a.parts, at = blockIdx.x / a.parts;
    const Item it = a.items[at];  // (of n_rows there may be)
    if (at >= *a.n_items) return;
    if ((unsigned) it.r >= (unsigned) a.n_rows || it.r0 < 0 || it.j < 0 || it.r0 + it.j != it.r || it.j >= it.n || it.r0 > a.n_rows - it.n || it.n > kMaxRows) return;
    RowState * const state = a.state + it.r;
    if (it.j > 0) {
        bool cut = it.parent < 0 || it.parent >= it.j;
        if (!cut) {
            const int next = agent_load(&a.state[it.r0 + it.parent].next);
            cut = next == kNone || next == kCut || (next >= 0 && next != it.j) || (next <= kFell && it.j <= kFell - next);
        }
        if (cut) {
            if (tid == 0) agent_store(&state->next, (int) kCut);
            return;
        }
    }
    const Rows w{it.r0, it.n};
    const bool greedy = !(it.t > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / (double) it.t;
    constexpr int E = NV * 4 * kT;
    const int i0 = part * E + 4 * tid;
    float x[NV][4], y[NV][4];
#pragma unroll
    for (int k = 0; k < NV; k++) values<4>(a.logits + it.r * a.ld, i0 + 4 * kT * k, a.V, a.vec, x[k]);
    const bool drawn = a.draft && !greedy && it.child < w.n;
    if (drawn)
#pragma unroll
        for (int k = 0; k < NV; k++) values<4>(a.draft + it.r * a.draft_ld, i0 + 4 * kT * k, a.V, a.vec, y[k]);
    Children kids{};
    if (wave == 0 && it.child < w.n) kids = children(a, w, it.j, it.j + 1);
    if (tid < 16) roots[tid] = a.roots[tid];
    float mp = -INFINITY, mq = -INFINITY;
    int top = 0x7fffffff;
    if (greedy) {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) argmax_take(mp, top, x[k][e] > 3.402823466e38f ? 3.402823466e38f : x[k][e], i0 + 4 * kT * k + e);
        for (int o = 32; o > 0; o >>= 1) argmax_take(mp, top, __shfl_xor(mp, o, 64), __shfl_xor(top, o, 64));
    } else {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) mp = fmaxf(mp, x[k][e]);
        mp = wave_max(mp);
        if (drawn) {
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) mq = fmaxf(mq, y[k][e]);
            mq = wave_max(mq);
        }
    }
    if (lane == 0) redm[0][wave] = mp, redm[1][wave] = mq, redt[wave] = top;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kT / 64; v++) {
        if (greedy) argmax_take(mp, top, redm[0][v], redt[v]);
        else mp = fmaxf(mp, redm[0][v]), mq = fmaxf(mq, redm[1][v]);
    }
    mp = fminf(mp, 3.402823466e38f);
    mq = fminf(mq, 3.402823466e38f);
    double sp = 0.0, sq = 0.0;
    if (!greedy) {
        const Soft p = soft(roots, inv_t, mp, 0.0), q = soft(roots, inv_t, mq, 0.0);
        if (mp > -INFINITY)
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) sp += p.weight(x[k][e]);
        if (drawn && mq > -INFINITY)
#pragma unroll
            for (int k = 0; k < NV; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) sq += q.weight(y[k][e]);
        sp = wave_sum_d(sp);
        sq = wave_sum_d(sq);
        if (lane == 0) red[0][wave] = sp, red[1][wave] = sq;
        __syncthreads();
        sp = sq = 0.0;
#pragma unroll
        for (int v = 0; v < kT / 64; v++) sp += red[0][v], sq += red[1][v];
    }
    PartSums * const sums = a.sums + (int64_t) it.r * a.parts;
    if (tid == 0) share(sums + part, PartSums{sp, sq, mp, mq, top, 0});
    if (!last_of(&state->arrived, a.parts, &flag) || wave) return;

    RowState z{0.0, 0.0, 0.0, -INFINITY, -INFINITY, 0x7fffffff, kNone, 0};
    const PartSums mine = lane < a.parts ? shared(sums + lane) : PartSums{0.0, 0.0, -INFINITY, -INFINITY, 0x7fffffff, 0};
    const auto each = [&](auto && f) {
        f(mine);
        for (int i = lane + 64; i < a.parts; i += 64) f(shared(sums + i));
    };
    each([&](const PartSums & x) {
        argmax_take(z.m_p, z.top, x.m_p, x.top);
        z.m_q = fmaxf(z.m_q, x.m_q);
    });
    for (int o = 32; o > 0; o >>= 1) argmax_take(z.m_p, z.top, __shfl_xor(z.m_p, o, 64), __shfl_xor(z.top, o, 64));
    z.m_q = wave_max(z.m_q);
    Soft p = soft(roots, inv_t, z.m_p, 0.0), q = soft(roots, inv_t, z.m_q, 0.0);
    if (!greedy) {
        each([&](const PartSums & x) {
            if (x.p > 0.0) z.sum_p += x.p * p.weight(x.m_p);
            if (x.q > 0.0) z.sum_q += x.q * q.weight(x.m_q);
        });
        z.sum_p = wave_sum_d(z.sum_p);
        z.sum_q = wave_sum_d(z.sum_q);
        p = soft(roots, inv_t, z.m_p, z.sum_p);
        q = soft(roots, inv_t, z.m_q, z.sum_q);
    }
    if (z.m_p > -INFINITY && it.child < w.n) {
        if (greedy) {
            for (int j0 = it.j + 1; j0 < w.n; kids = children(a, w, it.j, j0)) {
                const uint64_t hit = __ballot((kids.at >> lane & 1) && kids.token == z.top);
                if (hit) z.next = j0 + __builtin_ctzll(hit);
                if (hit || (j0 += 64) >= w.n) break;
            }
        } else if (drawn) decide_drawn(a, w, it.j, it.j, 1.0, p, q, kids, it.j + 1, z);
        else z.next = decide_guessed(a, w, it.j, p, kids);
    }
    if (lane == 0) {
        state->sum_p = z.sum_p, state->sum_q = z.sum_q, state->C = z.C, state->m_p = z.m_p, state->m_q = z.m_q, state->top = z.top;
        agent_store(&state->next, z.next);
    }
}

// The walk of one sequence. A part of the last row's weights w_k is a workgroup's, their sum for the draw or for the next child; the last
// workgroup to end goes on, in the last launch alone to the end.
__global__ __launch_bounds__(kT) void k_verify_walk(const VerifyArgs a) {
    constexpr int E = kDraw * kT;
    __shared__ double roots[16], red[2][kT / 64];
    __shared__ int next[kMaxRows], path[kMaxRows];
    __shared__ uint32_t gone[E / 32];
    __shared__ int flag, n_path, said;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = blockIdx.x / a.draws;
    if (a.seq[s].done) return;
    const Rows w = rows_of(a.starts, s, a.n_rows, a.max_rows);
    const float t = a.temperature ? a.temperature[s] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / (double) t;
    if (tid < 16) roots[tid] = a.roots[tid];
    bool alone = false;
    for (;;) {
        // the path as far as it is known
        for (int j = tid; j < w.n; j += kT) next[j] = a.state[w.r0 + j].next;
        __syncthreads();
        if (tid == 0) {
            int n = 0;
            for (int u = 0; w.n > 0 && n < a.max_path;) {
                path[n++] = u;
                if (next[u] <= u || next[u] >= w.n) break;
                u = next[u];
            }
            n_path = n;
        }
        __syncthreads();
        const int n = n_path, u = n ? path[n - 1] : 0;
        const RowState z = n ? a.state[w.r0 + u] : RowState{};
        const bool fell = z.next <= kFell, draw = n && (z.next == kNone || fell) && z.m_p > -INFINITY && !greedy;
        int token = -1;
        if (!draw) {
            if (!alone && blockIdx.x % a.draws) return;
            if (n && z.next >= 0 && z.next < w.n) token = a.tokens[w.r0 + z.next];  // (a path cut short)
            else if (n && greedy && z.m_p > -INFINITY) token = z.top;
        } else {
            const Soft p = soft(roots, inv_t, z.m_p, z.sum_p), q = soft(roots, inv_t, z.m_q, z.sum_q);
            const float * x = a.logits + (w.r0 + u) * a.ld, * y = a.draft + (w.r0 + u) * a.draft_ld;
            // the weights of the part's tokens i .. that this thread has; all: of r, the guesses that fell taken out, or of p
            const auto weights = [&](int part, bool all, double (&v)[kDraw], double & sum_w, double & sum_p) {
                const int i = part * E + kDraw * tid;
                float l[kDraw];
                values<kDraw>(x, i, a.V, a.vec, l);
                uint32_t out = 0;
                if (!a.draft) {
                    for (int b = tid; b < E / 32; b += kT) gone[b] = 0;
                    __syncthreads();
                    for (int j = u + 1 + tid; j < w.n; j += kT)
                        if (a.parents[w.r0 + j] == u) {
                            const unsigned e = (unsigned) a.tokens[w.r0 + j] - (unsigned) (part * E);
                            if (e < (unsigned) E) atomicOr(&gone[e / 32], 1u << (e % 32));
                        }
                    __syncthreads();
                    out = gone[tid * kDraw / 32] >> (tid * kDraw % 32);
                }
                sum_w = sum_p = 0.0;
                float d[kDraw];
                if (z.C > 0.0) values<kDraw>(y, i, a.V, a.vec, d);
#pragma unroll
                for (int e = 0; e < kDraw; e++) {
                    const double pe = p.p(l[e]);
                    v[e] = all ? pe : out >> e & 1 ? 0.0 : z.C > 0.0 ? fmax(pe - z.C * q.p(d[e]), 0.0) : pe;
                    sum_w += v[e];
                    sum_p += pe;
                }
            };
            Drawn * const drawn = a.drawn + (int64_t) s * a.draws;
            double v[kDraw];
            for (int part = alone ? 0 : blockIdx.x % a.draws; part < a.draws; part++) {
                double sw, sp;
                weights(part, false, v, sw, sp);
                sw = wave_sum_d(sw);
                sp = wave_sum_d(sp);
                if (lane == 0) red[0][wave] = sw, red[1][wave] = sp;
                __syncthreads();
                if (tid == 0) {
                    sw = sp = 0.0;
                    for (int i = 0; i < kT / 64; i++) sw += red[0][i], sp += red[1][i];
                    share(drawn + part, Drawn{sw, sp});
                }
                __syncthreads();
                if (!alone) break;
            }
            if (!alone && !last_of(&a.seq[s].arrived, a.draws, &flag)) return;
            // the parts' sums up to each one's, 64 parts at a time
            const Drawn mine64 = lane < a.draws ? shared(drawn + lane) : Drawn{};
            const auto part_of = [&](int i0) { return i0 ? (i0 + lane < a.draws ? shared(drawn + i0 + lane) : Drawn{}) : mine64; };
            const auto upto = [&](double v) {
                for (int o = 1; o < 64; o <<= 1) {
                    const double b = __shfl_up(v, o, 64);
                    if (lane >= o) v += b;
                }
                return v;
            };
            const auto sum_of = [&](bool all) {
                double sum = 0.0;
                for (int i0 = 0; i0 < a.draws; i0 += 64) {
                    const Drawn d = part_of(i0);
                    sum += readlane_d(upto(all ? d.p : d.w), 63);
                }
                return sum;
            };
            double total = sum_of(false);
            if (fell) {
                if (wave == 0) {
                    RowState o = z;
                    const int from = kFell - z.next, j0 = from + 1;
                    decide_drawn(a, w, u, from, total, p, q, children(a, w, u, j0), j0, o);
                    if (lane == 0) a.state[w.r0 + u].C = o.C, a.state[w.r0 + u].next = o.next;
                }
                if (!a.last) {
                    if (tid == 0) a.seq[s].arrived = 0;
                    return;
                }
                alone = true;
                __syncthreads();
                continue;
            }
            // the part, the thread, the token where the cumulative sum passes the coin's share
            const bool all = !(total > 0.0);
            if (all) total = sum_of(true);
            const float coin = a.coins[w.r0];
            const double want = (coin > 0.0f ? fmin((double) coin, 1.0 - 0x1p-24) : 0.0) * total;
            int part = 0;
            double base = 0.0, below = 0.0;
            for (int i0 = 0; i0 < a.draws; i0 += 64) {
                const Drawn x = part_of(i0);
                const double d = all ? x.p : x.w, sum = upto(d);
                const uint64_t some = __ballot(d > 0.0), hit = __ballot(d > 0.0 && below + sum > want);
                if (some) {  // (the last one with a weight, if rounding leaves no other)
                    const int l = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
                    part = i0 + l;
                    base = l ? below + readlane_d(sum, l - 1) : below;
                }
                if (hit) break;
                below += readlane_d(sum, 63);
            }
            double mine, sp;
            weights(part, all, v, mine, sp);
            if (all) mine = sp;
            const double sums = upto(mine);
            if (lane == 63) red[0][wave] = sums;
            if (tid == 0) flag = kT, said = -1;
            __syncthreads();
            for (int i = 0; i < wave; i++) base += red[0][i];
            if (mine > 0.0) {
                if (base + sums > want) atomicMin(&flag, tid);
                atomicMax(&said, tid);
            }
            __syncthreads();
            const int who = flag < kT ? flag : said;  // (rounding may leave none: the last one)
            __syncthreads();
            if (tid == who) {
                double c = base + (sums - mine);
                int e0 = 0;
                for (int e = 0; e < kDraw; e++)
                    if (v[e] > 0.0) {
                        e0 = e;
                        c += v[e];
                        if (c > want) break;
                    }
                said = part * E + kDraw * tid + e0;
            }
            __syncthreads();
            token = said;
        }
        int32_t * const rows = a.rows + (int64_t) s * a.max_path, * const out = a.out + (int64_t) s * a.max_path;
        for (int i = tid; i < a.max_path; i += kT) {
            rows[i] = i < n ? path[i] : -1;
            out[i] = i + 1 < n ? a.tokens[w.r0 + path[i + 1]] : i < n ? token : -1;
        }
        if (tid == 0) a.count[s] = n, a.seq[s].done = 1;
        return;
    }
}

// How a call is cut: values of a workgroup, and of a draw's.
struct VerifyShape {
    int nv, parts, draws;
    size_t items, state, sums, seq, drawn, total;  // offsets
};
VerifyShape verify_shape(int n_seq, int64_t n_rows, int64_t V) {
    VerifyShape z{};
    z.nv = n_rows * ((V + 8191) / 8192) >= 1024 ? 8 : 2;
    z.parts = (int) ((V + z.nv * 4 * kT - 1) / (z.nv * 4 * kT));
    z.draws = (int) ((V + kDraw * kT - 1) / (kDraw * kT));
    z.items = 256;
    z.state = z.items + align256((size_t) n_rows * sizeof(Item));
    z.sums = z.state + align256((size_t) n_rows * sizeof(RowState));
    z.seq = z.sums + align256((size_t) n_rows * z.parts * sizeof(PartSums));
    z.drawn = z.seq + align256((size_t) n_seq * sizeof(SeqState));
    z.total = z.drawn + align256((size_t) n_seq * z.draws * sizeof(Drawn));
    return z;
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
    return verify_shape(n_seq, n_rows, V).total;
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
        const VerifyShape z = verify_shape(n_seq, n_rows, n_vocab);
        uint8_t * const at = (uint8_t *) ws;
        VerifyArgs a{};
        a.starts = starts, a.parents = parents, a.tokens = tokens, a.logits = logits, a.ld = ld, a.draft = draft_logits, a.draft_ld = draft_ld;
        a.temperature = temperature, a.coins = coins, a.n_seq = n_seq, a.n_rows = (int) n_rows, a.V = (int) n_vocab;
        a.max_rows = (int) std::min<int64_t>(max_rows, std::max<int64_t>(n_rows, 1)), a.max_path = max_path;
        a.parts = z.parts, a.draws = z.draws;
        a.vec = aligned(logits, 16) && ld % 4 == 0 && (!draft_logits || (aligned(draft_logits, 16) && draft_ld % 4 == 0));
        a.count = count, a.rows = rows, a.out = tokens_out;
        a.n_items = (int *) at, a.items = (Item *) (at + z.items), a.state = (RowState *) (at + z.state);
        a.sums = (PartSums *) (at + z.sums), a.seq = (SeqState *) (at + z.seq), a.drawn = (Drawn *) (at + z.drawn);
        for (int i = 0; i < 16; i++) a.roots[i] = std::exp2(i / 16.0);
        hipStream_t st = as_stream(stream);
        k_verify_begin<<<paged_grid(std::max<int64_t>((n_rows + 3) / 4, 1), kT), kT, 0, st>>>(a);
        check_launch("draft verify");
        if (n_rows) {
            const unsigned grid = paged_grid(n_rows * z.parts, kT);
            if (z.nv == 8) k_verify_rows<8><<<grid, kT, 0, st>>>(a);
            else k_verify_rows<2><<<grid, kT, 0, st>>>(a);
            check_launch("draft verify rows");
        }
        // A path that cannot be all of a sequence's rows tells that rows have several children, of which some will fall.
        for (int left = draft_logits && max_path < a.max_rows && z.draws > 4 ? 3 : 1; left; left--) {
            a.last = left == 1;
            k_verify_walk<<<paged_grid((int64_t) n_seq * z.draws, kT), kT, 0, st>>>(a);
            check_launch("draft verify walk");
        }
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
