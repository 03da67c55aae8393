// draft.hip - steps with drafted tokens: the trees' masks and positions, the drafts' verification, and moving the accepted rows
// together in the caches (include/gcq_draft.h; append and attention of such rows are paged.hip's and paged_attn.hip's).
#include <algorithm>
#include <vector>

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
// 1024 rows fit. Latency, a few rounds in LDS: a tree of 26 rows 4 us, 64 trees of 40 to 255 rows 8.
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
// k_verify_begin puts the rows in order, the sequences' first rows first, then their second ones, .. k_verify_rows takes each row's logits
// in parts, a workgroup to a part: the largest and the sum of exponentials, of the target's and, where a row has children, the
// drafter's. Whichever of a row's workgroups ends last has the row's softmax and decides which child stands, which depends on
// nothing but the row. Rows that an earlier decision has cut off from the path are passed over if it is known by then: in this
// order, where rows are many, it mostly is (nobody waits for it, and no result depends on it). The decision that completes a path
// from the root puts it out and leaves the last row to k_verify_draw, which draws its token. Where drawn children fell it is drawn
// from what they left:
//   r after k fallen drafts is w_k / c_k, w_k = max(p - C_k q, 0), c_k its sum, C_0 = 0 and C_k+1 = C_k + c_k, since
//   max(max(a, 0) - b, 0) = max(a - b, 0) for b >= 0: one sum over the vocabulary for each that falls, made for the rows on the
//   path alone.
//
// In 64 bits: a token's border in the cumulative sum would be off by 2^-25 or so in 32, and 10^5 borders then put a drawn token wrong
// once in some hundred draws.

typedef int i4_t __attribute__((ext_vector_type(4)));

constexpr int kT = 256, kStep = 4 * kT;  // threads, logits of a workgroup at a time
constexpr int kSteps = 8;                // .. of a part at most
constexpr int kDrawT = 512;              // threads of k_verify_draw
constexpr int kRowGroups = 768;          // workgroups at a time in k_verify_rows: three on a CU (64 chains 88 us, 99 with four; 16 trees 59 and 64)
constexpr int kApart = 64;               // ints from one row's counter to the next: in one line all rows' workgroups queue, some 8 ns each (64 single rows 34 us, 31 so)
constexpr float kHuge = 3.402823466e38f;

// What became of a row: the child that stands (>= 0), or
enum : int { kNone = -1, kOpen = -2, kLeft = -3, kFell = -16 };  // not known yet; all drawn ones fell; kFell - j: child j fell, others are left

struct __align__(16) RowState {
    double sum_p, sum_q, C;  // sums of exp((l - m) / t)
    float m_p, m_q;
    int top, pad;
};
struct __align__(16) PartSums {
    double p, q;
    float m_p, m_q;
    int top, pad;
};
struct __align__(16) SeqState {  // a sequence whose path is known
    int u, n, then, r0;            // the path's last row, its rows (0: not known, or ended), what became of it; the sequence's rows
    int rows, arrived, listed;       // listed: it draws from what is left; not changed behind k_verify_rows
    float t;
};
struct __align__(16) Item {  // a row in its order
    int r, s, j, parent;  // parent < 0: none
    int r0, n;            // its sequence's rows
    float t;              // temperature
    int child;            // the first; n: none
};

struct VerifyArgs {
    const int32_t * starts, * parents, * tokens;
    const float * logits, * draft, * temperature, * coins;
    int64_t ld, draft_ld;
    int n_seq, n_rows, V, max_rows, max_path;
    int parts, steps, abreast, blocks, block_steps;  // parts of a row and a part's steps; rows abreast in k_verify_rows; parts of what is left
    bool vec, last;                     // rows of whole 16-byte pieces; the last k_verify_draw
    int32_t * count, * rows, * out;
    int * n_items, * n_list, * list;  // the sequences that draw from what is left
    Item * items;
    RowState * state;
    int * next, * arrived;  // of the rows (arrived kApart apart)
    PartSums * sums;
    SeqState * seq;
    double * drawn, * drawn_runs;  // of a sequence's parts of what is left, and of their runs of 256 tokens
};

// 2^(i / 32), i of 32, its bits i 2^47 less: with n 2^47 more root n % 32 is 2^(n / 32).
__device__ __forceinline__ double root_of(int i) {
    const double y = exp2(i * 0x1p-5);
    return __hiloint2double(__double2hiint(y) - (i << 15), __double2loint(y));
}

// exp by a 32nd of a power of two from LDS and four terms of exp's series on what is left, the fifth taken into the others
// (z^5 = 5/4 a^2 z^3 - 5/16 a^4 z but for a^5 / 16, |z| <= a = ln 2 / 64: 2^-43). 11 operations of 64 bits and 4 others in `weigh4`, where the
// kernels spend their arithmetic; the library's takes some 30. (Loops are left as loops here, and code is written once: most of it
// runs once in a workgroup, and fetching 40 KB of it took longer than what it did.)
__device__ __forceinline__ double power(double r) {  // 2^(r / 32), |r| <= 1 / 2
    constexpr double k = 0.021660849392498290;           // ln 2 / 32
    constexpr double c5 = k * k * k * k * k / 120;
    double y = fma(r, k * k * k * k / 24, k * k * k / 6 + c5 * 0.3125);
    y = fma(r, y, k * k / 2);
    y = fma(r, y, k - c5 * 0.01953125);
    return fma(r, y, 1.0);
}
// 2^(n / 32)
__device__ __forceinline__ double root(const double * roots, int n) {
    const double y = roots[n & 31];
    return __hiloint2double(__double2hiint(y) + (n << 15), __double2loint(y));
}
struct Soft {
    const double * roots;  // LDS
    double scale, m, inv;  // 32 / (t ln 2); a logit that weighs 1, the row's weights are below 2^512; 1 / their sum
    // exp((l - m) / t), 0 from 2^-1000 on
    __device__ __forceinline__ double weight(float l) const {
        if (l > kHuge) l = kHuge;
        const double x = ((double) l - m) * scale, t = x + 0x1.8p52, y = power(x - (t - 0x1.8p52)) * root(roots, (int) (uint32_t) __double_as_longlong(t));
        return x > -32000.0 ? y : 0.0;  // (nor for -inf and NaN)
    }
    __device__ __forceinline__ double p(float l) const { return weight(l) * inv; }
};
__device__ __forceinline__ double scale_of(float t) { return 46.166241308446828 / (double) t; }
__device__ __forceinline__ Soft soft(const double * roots, double scale, float m, double sum) { return {roots, scale, (double) m, sum > 0.0 ? 1.0 / sum : 0.0}; }

// Logits around m where the short form serves: those above `low` (2^-1000; what is below counts as that, no more than 2^-1000 each, NaN too),
// and not above `high`, 2^500; -inf if there is no such range in f32, or no such m.
struct Range {
    float low, high;
};
__device__ __forceinline__ Range range_of(float m, double scale) {
    const double d = 32000.0 / scale;
    const Range z{(float) ((double) m - d), (float) ((double) m + 0.5 * d)};
    const double x = ((double) z.low - (double) m) * scale;
    const bool odd = !(fabsf(m) < 1e38f) || !(x > -32600.0 && x < -31400.0);  // (root's powers end at 2^-1022)
    return {z.low, odd ? -INFINITY : z.high};
}
// A NaN as one that maxima and medians pass over (a signalling one comes out of them).
__device__ __forceinline__ float quiet(float l) { return __builtin_canonicalizef(l); }
// The weights of four logits in that range (two, then two: more at a time than the registers hold).
__device__ __forceinline__ void weigh4(const double * roots, double scale, double m, float low, const float (&l)[4], double (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
#pragma unroll
        for (int i = e; i < e + 2; i++) {
            const double d = (double) __builtin_amdgcn_fmed3f(quiet(l[i]), low, kHuge) - m, t = fma(d, scale, 0x1.8p52), r = fma(d, scale, 0x1.8p52 - t);
            v[i] = power(r) * root(roots, (int) (uint32_t) __double_as_longlong(t));
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// A sum of weights; m: the logit that weighs 1, -inf while there is none.
struct Running {
    float m;
    double s;
    // s2 times exp(m2 / t) more
    __device__ __forceinline__ void take(const double * roots, double scale, float m2, double s2) {
        if (!__any(m > -INFINITY)) {
            m = m2, s = s2;
            return;
        }
        const Soft z{roots, scale, (double) fmaxf(m, m2), 0.0};
        s = s * z.weight(m) + s2 * z.weight(m2);
        m = fmaxf(m, m2);
    }
    // in: m's, at first {0, -inf}
    __device__ __forceinline__ void take4(const double * roots, double scale, Range & in, const float (&l)[4]) {
        const float top = fmaxf(fmaxf(quiet(l[0]), quiet(l[1])), fmaxf(quiet(l[2]), quiet(l[3])));  // (NaNs passed over)
        if (__any(top > in.high)) {
            if (m == -INFINITY && top > -INFINITY) {
                m = fminf(top, kHuge), s = 0.0;
                in = range_of(m, scale);
            }
            if (__any(top > in.high)) {
                const float to = fminf(fmaxf(m, top), kHuge);
                if (to > -INFINITY) {
                    const Soft z{roots, scale, (double) to, 0.0};
                    s *= z.weight(m);
                    m = to;
                    in = range_of(m, scale);
                    float x = l[0], y = l[1], u = l[2], v = l[3];
#pragma unroll 1
                    for (int e = 0; e < 4; e++) {
                        s += z.weight(x);
                        x = y, y = u, u = v;
                    }
                }
                return;
            }
        }
        double v[4];
        weigh4(roots, scale, m > -INFINITY ? (double) m : 0.0, in.low, l, v);
        const double more = (v[0] + v[1]) + (v[2] + v[3]);
        s += top > -INFINITY ? more : 0.0;  // (there may be no m yet, or no short form)
    }
    __device__ __forceinline__ void wave(const double * roots, double scale) {
        const float top = wave_max(m);
        s = wave_sum_d(m > -INFINITY ? s * Soft{roots, scale, (double) top, 0.0}.weight(m) : 0.0);
        m = top;
    }
};

// Four values x[i ..), those at V and beyond -inf; whole: there are none of those, and 16-byte pieces.
__device__ __forceinline__ void values4(const float * x, int i, int V, bool whole, float (&v)[4]) {
    if (whole) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + i);
    else
#pragma unroll
        for (int c = 0; c < 4; c++) {
            v[c] = -INFINITY;
            if (i + c < V) v[c] = x[i + c];
        }
}

template <class T>
__device__ __forceinline__ T agent_load(const T * p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T>
__device__ __forceinline__ void agent_store(T * p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// What workgroups tell each other within a launch goes past the XCDs' L2s, word by word, and a store that others go by follows once what came
// before has reached memory: a fence would write back and drop a whole L2, some 40 ns each and one after the other.
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
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Whether this workgroup is the last of n to arrive, after thread 0 has shared what it has (all threads together).
__device__ __forceinline__ bool last_of(int * arrived, int n, int * flag) {
    if (threadIdx.x == 0) {
        stores_done();
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

// A wavefront to a row: its place in the order, and its state. Latency: 5 rows 2.6 us, 800 rows of 16 trees 4.9, of 1024 sequences, which it looks
// through 64 at a time, 10.
__global__ __launch_bounds__(kT) void k_verify_begin(const VerifyArgs a) {
    const int lane = threadIdx.x & 63, r = blockIdx.x * (kT / 64) + (threadIdx.x >> 6);
    const int64_t id = (int64_t) blockIdx.x * kT + threadIdx.x, all_ids = (int64_t) gridDim.x * kT;  // (64 threads a row: from 2^25 rows on past 31 bits)
    if (id == 0) *a.n_list = 0;
    for (int64_t s = id; s < a.n_seq; s += all_ids) a.seq[s] = SeqState{}, a.count[s] = 0;
    for (int64_t i = id; i < (int64_t) a.n_seq * a.max_path; i += all_ids) a.rows[i] = a.out[i] = -1;
    if (r >= a.n_rows) return;
    if (lane == 0) a.next[r] = kOpen, a.arrived[(int64_t) r * kApart] = 0;
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
        if (lane == 0) *a.n_items = min(all, a.n_rows);
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
// Whether the child at bit l of k, the children from row j0 on, has the token of an earlier one.
__device__ __forceinline__ bool again(const VerifyArgs & a, const Rows & w, int u, const Children & k, int j0, int l, int token) {
    const int lane = threadIdx.x & 63;
    bool before = (k.at >> lane & 1) && lane < l && k.token == token;
    for (int i = u + 1 + lane; i < j0; i += 64) before = before || (a.parents[w.r0 + i] == u && a.tokens[w.r0 + i] == token);
    return __any(before);
}
// Which of row u's children after row `from` stands (a wavefront; k: its children from row j0 on): the first with the largest logit's token
// (top >= 0); of drawn ones the next, c being r's sum; of guesses the first that stands, c what is left of p.
__device__ __forceinline__ int decide(const VerifyArgs & a, const Rows & w, int u, int from, int top, double c, const Soft & p, const Soft & q,
                                      Children k, int j0, double & C) {
    for (;;) {
        const int lane = threadIdx.x & 63;
        uint64_t at = __ballot((k.at >> lane & 1) && j0 + lane > from && (top < 0 || k.token == top));
        if (top >= 0 && at) return j0 + __builtin_ctzll(at);
        const double pt = p.p(k.x), qt = a.draft ? q.p(k.y) : 1.0;  // (0 of a token that there is not)
        for (; at; at &= at - 1) {
            const int l = __builtin_ctzll(at);
            const double ql = readlane_d(qt, l);
            double v = readlane_d(pt, l);
            if (a.draft) v = fmax(v - C * ql, 0.0);
            else if (again(a, w, u, k, j0, l, __builtin_amdgcn_readlane(k.token, l))) v = 0.0;
            if ((double) readlane_f(k.coin, l) * c * ql < v) return j0 + l;
            if (a.draft) {
                C += c;
                return at & (at - 1) || child_after(a.parents, w, u, j0 + 63) < w.n ? kFell - (j0 + l) : (int) kLeft;
            }
            c -= v;
        }
        if ((j0 += 64) >= w.n) return kNone;
        k = children(a, w, u, j0);
    }
}

// What a workgroup keeps in LDS for a draw.
struct DrawLds {
    double roots[32], seg[4 * kSteps];  // sums of a part's runs of 256 tokens
    uint32_t gone[kSteps * kStep / 32];
    int flag, said;
};

// The path on from row u, its row n (a wavefront): its rows, the last one and what became of that; on: `row` is one of them. PUT: into the results.
struct Path {
    int n, u, then;
    bool on;
    int mine;  // a lane's of its last rows, those of one 64
};
// Rows first .. n - 1 of a path, a lane's each, and that each follows the one before.
__device__ __forceinline__ void put_rows(const VerifyArgs & a, const Rows & w, int s, int first, int n, int row) {
    const int i = first + (threadIdx.x & 63);
    if (i >= n) return;
    a.rows[(int64_t) s * a.max_path + i] = row;
    if (i) a.out[(int64_t) s * a.max_path + i - 1] = a.tokens[w.r0 + row];
}
template <bool PUT>
__device__ __forceinline__ Path follow(const VerifyArgs & a, const Rows & w, int s, int n, int u, int row) {
    const int lane = threadIdx.x & 63;
    Path z{n, u, kOpen, false, 0};
    int at = -1, next = kOpen, first = n;
    const auto put = [&] {
        if (PUT) put_rows(a, w, s, first, z.n, z.mine);
    };
    for (;;) {
        if (lane == ((z.n - first) & 63)) z.mine = z.u;
        z.on = z.on || z.u == row;
        z.n++;
        if (PUT && z.n - first == 64) put(), first = z.n;
        if (z.u >> 6 != at) {
            at = z.u >> 6;
            next = agent_load(&a.next[w.r0 + min(64 * at + lane, w.n - 1)]);
        }
        z.then = __builtin_amdgcn_readlane(next, z.u & 63);
        if (z.then <= z.u || z.then >= w.n || z.n >= a.max_path) break;
        z.u = z.then;
    }
    put();
    return z;
}

// A lane's value and those of the lanes before.
__device__ __forceinline__ double upto(double v) {
    const auto add = [&](auto move) { v += __hiloint2double(move(__double2hiint(v)), move(__double2loint(v))); };
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true); });  // row_shr 1, 2, 4, 8
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true); });
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); });  // lane 15 into the next row, then 31 into the upper half
    add([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); });
    return v;
}

// A row that a token is drawn from: its r, max(p - C q, 0) if C > 0, else p without the guesses that fell.
struct Source {
    Rows w;
    int s, u;
    double C;
    Soft p, q;
    float p_low, q_low;  // Range's
    bool odd;
    int parts, steps;
};
__device__ __forceinline__ Source source(const VerifyArgs & a, const Rows & w, int s, int u, const RowState & st, const double * roots, double scale) {
    const Range p = range_of(st.m_p, scale), q = st.C > 0.0 ? range_of(st.m_q, scale) : p;
    return {w, s, u, st.C, soft(roots, scale, st.m_p, st.sum_p), soft(roots, scale, st.m_q, st.sum_q), p.low, q.low, !(p.high > -INFINITY && q.high > -INFINITY),
            st.C > 0.0 ? a.blocks : a.parts, st.C > 0.0 ? a.block_steps : a.steps};
}
// The weights of the tokens whose logits are l (the drafter's d), from token i of a part on, of r or (all) of p.
__device__ __forceinline__ void weights4(const VerifyArgs & a, const Source & z, const DrawLds & m, int i, bool all, const float (&l)[4], const float (&d)[4], double (&v)[4]) {
    const bool fell = z.C > 0.0 && !all;
    double q[4];
    if (z.odd) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = z.p.weight(l[e]);
            if (fell) q[e] = z.q.weight(d[e]);
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        weigh4(z.p.roots, z.p.scale, z.p.m, z.p_low, l, v);
        if (fell) weigh4(z.q.roots, z.q.scale, z.q.m, z.q_low, d, q);
    }
    const uint32_t out = a.draft || all ? 0 : m.gone[i / 32] >> (i % 32);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[e] = out >> e & 1 ? 0.0 : v[e] * z.p.inv;
        if (fell) v[e] = fmax(v[e] - z.C * (q[e] * z.q.inv), 0.0);
    }
}
__device__ __forceinline__ void logits4(const VerifyArgs & a, const Source & z, int part, int i, bool all, float (&l)[4], float (&d)[4]) {
    const int at = part * z.steps * kStep + i;
    const bool whole = a.vec && at + 3 < a.V;
    values4(a.logits + (z.w.r0 + z.u) * a.ld, at, a.V, whole, l);
    if (z.C > 0.0 && !all) values4(a.draft + (z.w.r0 + z.u) * a.draft_ld, at, a.V, whole, d);
}
// The sums of a part's runs of 256 tokens, and of the part (all threads).
__device__ __forceinline__ double runs(const VerifyArgs & a, const Source & z, DrawLds & m, int part, bool all) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (!a.draft && !all) {
        for (int i = tid; i < kSteps * kStep / 32; i += kDrawT) m.gone[i] = 0;
        __syncthreads();
        for (int j = z.u + 1 + tid; j < z.w.n; j += kDrawT)
            if (a.parents[z.w.r0 + j] == z.u) {
                const unsigned e = (unsigned) a.tokens[z.w.r0 + j] - (unsigned) (part * z.steps * kStep);
                if (e < (unsigned) (z.steps * kStep)) atomicOr(&m.gone[e / 32], 1u << (e % 32));
            }
        __syncthreads();
    }
    float l[4], d[4], l1[4], d1[4];
    logits4(a, z, part, 4 * tid, all, l, d);
#pragma unroll 1
    for (int i = 4 * tid; i < z.steps * kStep; i += 4 * kDrawT) {
        if (i + 4 * kDrawT < z.steps * kStep) logits4(a, z, part, i + 4 * kDrawT, all, l1, d1);
        double v[4];
        weights4(a, z, m, i, all, l, d, v);
#pragma unroll
        for (int e = 0; e < 4; e++) l[e] = l1[e], d[e] = d1[e];
        const double sum = wave_sum_d((v[0] + v[1]) + (v[2] + v[3]));
        if ((tid & 63) == 0) m.seg[i / 256] = sum;
    }
    __syncthreads();
    return wave_sum_d((tid & 63) < 4 * z.steps ? m.seg[tid & 63] : 0.0);
}
static_assert(4 * kSteps <= 64 && kStep % (4 * 64) == 0, "a run to a lane, whole runs");

// The sum of a lane's part, of those from i0 on: what fell of drawn ones was summed for this draw, others are k_verify_rows's (the first 64
// of them `early`), less what fell.
__device__ __forceinline__ double part_sum(const VerifyArgs & a, const Source & z, int i0, bool all, const PartSums & early) {
    const int lane = threadIdx.x & 63, part = i0 + lane;
    if (z.C > 0.0 && !all) return part < z.parts ? shared(a.drawn + (int64_t) z.s * z.parts + part) : 0.0;
    double v = 0.0;
    if (part < z.parts) {
        PartSums x = early;
        if (i0) x = a.sums[(int64_t) (z.w.r0 + z.u) * z.parts + part];
        v = x.p * z.p.p(x.m_p);
    }
    if (all || a.draft) return v;
    for (int j0 = z.u + 1; j0 < z.w.n; j0 += 64) {
        const Children k = children(a, z.w, z.u, j0);
        const double pt = z.p.p(k.x);
        for (uint64_t at = k.at; at; at &= at - 1) {
            const int l = __builtin_ctzll(at), token = __builtin_amdgcn_readlane(k.token, l);
            const bool first = !again(a, z.w, z.u, k, j0, l, token);  // (all lanes)
            if (first && token >= 0 && token / (z.steps * kStep) == part) v -= readlane_d(pt, l);
        }
    }
    return fmax(v, 0.0);
}
constexpr double kNothing = 0x1p-900;  // no token's weight
// Of 64 lanes' values d, their sums up to each one `sum`: the one where it passes `want`, the last above nothing if rounding leaves none, -1 if all are 0; below grows by those before
// it, or by all.
__device__ __forceinline__ int pass(double d, double sum, double want, double & below, bool & hit) {
    const uint64_t some = __ballot(d > kNothing), at = __ballot(d > kNothing && below + sum > want);
    hit = at != 0;
    const int l = hit ? __builtin_ctzll(at) : some ? 63 - __builtin_clzll(some) : -1;
    below += hit ? (l ? readlane_d(sum, l - 1) : 0.0) : readlane_d(sum, 63);
    return l;
}
// The token where the cumulative sum passes the coin's share of it: the part, the run, the lane, the token; -1 if there is no sum. all: of p, whatever fell.
__device__ __forceinline__ int draw(const VerifyArgs & a, const Source & z, DrawLds & m, bool all, const PartSums & early) {
    const int lane = threadIdx.x & 63;
    const float coin = a.coins[z.w.r0];
    double d = 0.0, sum = 0.0, want = INFINITY, base = 0.0, rest = 0.0;
    int part = -1;
    bool hit = false;
#pragma unroll 1
    for (int find = 0; find < 2; find++) {  // the total, then the part
        double below = 0.0;
        for (int i0 = 0; i0 < z.parts && !hit; i0 += 64) {
            const double before = below;
            if (!find || z.parts > 64) d = part_sum(a, z, i0, all, early), sum = upto(d);
            const int l = pass(d, sum, want, below, hit);
            if (find && l >= 0) part = i0 + l, base = hit ? below : before, rest = hit ? want : INFINITY;
        }
        want = (coin > 0.0f ? fmin((double) coin, 1.0 - 0x1p-24) : 0.0) * below;
    }
    if (part < 0) return -1;
    want = rest;  // (no part passes it, by rounding: the last token of the last)
    const bool fell = z.C > 0.0 && !all;
    if (!fell) runs(a, z, m, part, all);
    if (threadIdx.x < 64) {
        d = 0.0;
        if (lane < 4 * z.steps) d = fell ? shared(a.drawn_runs + ((int64_t) z.s * z.parts + part) * (4 * z.steps) + lane) : m.seg[lane];
        const int run = pass(d, upto(d), want, base, hit);
        int token = -1;
        if (run >= 0) {
            if (!hit) want = INFINITY;
            float x[4], y[4];
            double v[4];
            logits4(a, z, part, run * 256 + 4 * lane, all, x, y);
            weights4(a, z, m, run * 256 + 4 * lane, all, x, y, v);
            d = (v[0] + v[1]) + (v[2] + v[3]);
            const int who = pass(d, upto(d), want, base, hit);
            if (who >= 0) {
                if (!hit) want = INFINITY;
                int e = -1;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const double x = readlane_d(v[i], who);
                    if (x > kNothing && (e < 0 || !(base > want))) e = i;
                    base += x;
                }
                token = part * z.steps * kStep + run * 256 + 4 * who + e;
            }
        }
        if (lane == 0) m.said = token;
    }
    __syncthreads();
    return m.said;
}

// A workgroup has one part of every abreast-th row: those in work at a time are the next of the order that are not cut off. Four wavefronts
// read; the fifth meets them once for a part: it has then looked up the next row and this one's children, and shares the part's sums and,
// its row's last, decides while they read that. Bound by HBM, arithmetic in 64 bits and, at the end, what one row's decision takes (6 us): 64 chains of 128256 tokens, 149 MB,
// 55 us (47 without the fifth's work, 42 without arithmetic); 16 trees, where decisions follow each other, 73 MB, 37 us; one chain 10.
__global__ __launch_bounds__(kT + 64, 4) void k_verify_rows(const VerifyArgs a) {
    struct Met {
        Running p[kT / 64], q[kT / 64];
        int top[kT / 64];
        Item next;
    };
    __shared__ double roots[32];
    __shared__ Met met[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = blockIdx.x % a.parts;
    if (tid < 32) roots[tid] = root_of(tid);
    int rank = blockIdx.x / a.parts;
    Item it = a.items[rank];
    const int n_items = min(*a.n_items, a.n_rows);
    if (rank >= n_items) return;
    __syncthreads();
    const auto join = [&](bool greedy, bool drawn, double scale, Running & p, Running & q, int & top) {
        if (greedy) {
#pragma unroll 1
            for (int o = 32; o > 0; o >>= 1) argmax_take(p.m, top, __shfl_xor(p.m, o, 64), __shfl_xor(top, o, 64));
        } else {
            p.wave(roots, scale);
            if (drawn) q.wave(roots, scale);
        }
    };
    const auto good = [&](const Item & it) {  // (starts that do not ascend)
        return (unsigned) it.s < (unsigned) a.n_seq && it.r0 >= 0 && it.j >= 0 && it.r0 + it.j == it.r && it.j < it.n && it.r0 <= a.n_rows - it.n && it.n <= kMaxRows;
    };
    if (wave < kT / 64) {
        for (int turn = 0; good(it); turn ^= 1) {
            Met & now = met[turn];
            const bool greedy = !(it.t > 0.0f), drawn = a.draft && !greedy && it.child < it.n;
            const double scale = greedy ? 1.0 : scale_of(it.t);
            const float * const x = a.logits + it.r * a.ld, * const y = drawn ? a.draft + it.r * a.draft_ld : x;
            Running p{-INFINITY, 0.0}, q{-INFINITY, 0.0};
            Range p_in{0.0f, -INFINITY}, q_in{0.0f, -INFINITY};
            int top = 0x7fffffff, i0 = part * a.steps * kStep + 4 * tid;
            asm("" : "+v"(i0));  // (or every comparison with it is kept over the loop)
            const auto load = [&](int k, float (&l)[4], float (&d)[4]) {
                const bool whole = a.vec && (part * a.steps + k + 1) * kStep <= a.V;
                values4(x, i0 + k * kStep, a.V, whole, l);
                if (drawn) values4(y, i0 + k * kStep, a.V, whole, d);
            };
            const auto take = [&](int k, const float (&l)[4], const float (&d)[4]) {
                if (greedy) {
#pragma unroll
                    for (int e = 0; e < 4; e++) argmax_take(p.m, top, l[e] > kHuge ? kHuge : l[e], i0 + k * kStep + e);
                } else {
                    p.take4(roots, scale, p_in, l);
                    if (drawn) q.take4(roots, scale, q_in, d);
                }
            };
            float l[2][4], d[2][4];
            load(0, l[0], d[0]);
            load(1, l[1], d[1]);
#pragma unroll 1
            for (int k = 0; k < a.steps; k += 2) {  // (an even number)
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    take(k + b, l[b], d[b]);
                    if (k + b + 2 < a.steps) load(k + b + 2, l[b], d[b]);
                }
            }
            join(greedy, drawn, scale, p, q, top);
            if (lane == 0) now.p[wave] = p, now.q[wave] = q, now.top[wave] = top;
            __syncthreads();
            it = now.next;
        }
        return;
    }
    Item done{};
    Children kids{};  // done's
    for (int turn = 0;; turn ^= 1) {
        // the row before: its sums first of the wavefronts, then, for the last of the row's workgroups to end, of the parts
        const auto end = [&] {
            const Met & was = met[turn ^ 1];
            const Rows w{done.r0, done.n};
            const bool greedy = !(done.t > 0.0f), drawn = a.draft && !greedy && done.child < done.n;
            const double scale = greedy ? 1.0 : scale_of(done.t);
            PartSums * const sums = a.sums + (int64_t) done.r * a.parts;
            Running p, q;
            int top;
#pragma unroll 1
            for (int round = 0; round < 2; round++) {
                p = q = Running{-INFINITY, 0.0};
                top = 0x7fffffff;
                for (int i = lane; i < (round ? a.parts : kT / 64); i += 64) {
                    const PartSums z = round ? shared(sums + i) : PartSums{was.p[i].s, was.q[i].s, was.p[i].m, was.q[i].m, was.top[i], 0};
                    if (greedy) argmax_take(p.m, top, z.m_p, z.top);
                    else {
                        p.take(roots, scale, z.m_p, z.p);
                        if (drawn) q.take(roots, scale, z.m_q, z.q);
                    }
                }
                join(greedy, drawn, scale, p, q, top);
                if (round) break;
                int last = 0;
                if (lane == 0) {
                    share(sums + part, PartSums{p.s, q.s, p.m, q.m, top, 0});
                    stores_done();
                    last = __hip_atomic_fetch_add(a.arrived + (int64_t) done.r * kApart, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.parts - 1;
                }
                if (!__builtin_amdgcn_readfirstlane(last)) return;
            }
            double C = 0.0;
            int next = kNone;
            if (p.m > -INFINITY && done.child < done.n)
                next = decide(a, w, done.j, done.j, greedy ? top : -1, 1.0, soft(roots, scale, p.m, p.s), soft(roots, scale, q.m, q.s), kids, done.j + 1, C);
            if (lane == 0) {
                a.state[done.r] = RowState{p.s, q.s, C, p.m, q.m, top, 0};
                agent_store(&a.next[done.r], next);
            }
            // Whoever decides a path's last row to be decided sees the others' decisions, its own being known before they are looked at.
            Path path{1, 0, next, true, 0};
            if (done.j > 0 || next >= 0) {
                stores_done();
                path = follow<false>(a, w, done.s, 0, 0, done.j);
            }
            if (!path.on || path.then == kOpen || (path.then >= 0 && path.n < a.max_path)) return;
            SeqState & seq = a.seq[done.s];  // (two at once write the same)
            int listed = 1;
            if (path.then < kOpen && lane == 0) listed = __hip_atomic_exchange(&seq.listed, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (path.n <= 64) put_rows(a, w, done.s, 0, path.n, path.mine);
            else follow<true>(a, w, done.s, 0, 0, done.j);
            if (lane) return;
            a.count[done.s] = path.n;
            if (path.then >= 0) a.out[(int64_t) done.s * a.max_path + path.n - 1] = a.tokens[w.r0 + path.then];  // (cut short)
            else seq.u = path.u, seq.n = path.n, seq.then = path.then, seq.r0 = w.r0, seq.rows = w.n, seq.t = done.t;
            if (!listed) a.list[__hip_atomic_fetch_add(a.n_list, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)] = done.s;
        };
        if (done.n > 0) end();
        if (!good(it)) return;
        // the next row that no decision so far cuts off, 64 at a time
        // (as two vectors: an Item goes by way of an address, which is made from the launch packet, in the host's memory: 2 us, 15 where a
        // thousand workgroups do so)
        i4_t x = {}, y = {};  // r, s, j, parent; r0, n, t, child
        for (rank += a.abreast; rank < n_items; rank += 64 * a.abreast) {
            const int mine = rank + lane * a.abreast;
            bool on = mine >= rank && mine < n_items;
            if (on) {
                x = reinterpret_cast<const i4_t *>(a.items + mine)[0], y = reinterpret_cast<const i4_t *>(a.items + mine)[1];
                on = x.z == 0 || x.w >= 0;
                for (int c = x.z, u = x.w; on && u >= 0 && u < c && c < kMaxRows && y.x >= 0 && y.x < a.n_rows - c;) {
                    const int next = agent_load(&a.next[y.x + u]), up = a.parents[y.x + u];
                    on = next == kOpen || next == c || (next <= kFell && c > kFell - next);
                    c = u, u = up;
                }
            }
            const uint64_t at = __ballot(on);
            if (at) {
                const int l = __builtin_ctzll(at);
                rank += l * a.abreast;
                if (lane == l) reinterpret_cast<i4_t *>(&met[turn].next)[0] = x, reinterpret_cast<i4_t *>(&met[turn].next)[1] = y;
                break;
            }
        }
        if (rank >= n_items && lane == 0) met[turn].next.n = -1, met[turn].next.j = 0;
        kids.at = 0;
        if (it.child < it.n) kids = children(a, Rows{it.r0, it.n}, it.j, it.j + 1);
        __syncthreads();
        done = it;
        it = met[turn].next;
    }
}

// The last rows' tokens: of p by workgroup s, from k_verify_rows's sums; of what drawn children left a workgroup a part, which it sums, for the
// draw or for the next child: the last of the sequence's to end goes on, in the last launch alone to the path's end.
// Bound by its depth, a few us for a sum, then total, part, run and token, 1 to 2 us each: one chain 10 us, 64 chains 17.5 (24 MB), 16 trees' guesses 10.
__global__ __launch_bounds__(kDrawT) void k_verify_draw(const VerifyArgs a) {
    __shared__ DrawLds m;
    __shared__ Path path;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < 32) m.roots[tid] = root_of(tid);
    const bool of_p = (int) blockIdx.x < a.n_seq;
    const int units = of_p ? a.n_seq : min(*a.n_list, a.n_seq) * a.blocks;
    for (int unit = of_p ? blockIdx.x : blockIdx.x - a.n_seq; unit < units; unit += of_p ? a.n_seq : gridDim.x - a.n_seq) {
        const int s = of_p ? unit : a.list[unit / a.blocks], own = unit % a.blocks;
        if ((unsigned) s >= (unsigned) a.n_seq) return;
        const SeqState & q = a.seq[s];
        const Rows w{q.r0, q.rows};
        const float t = q.t;
        int u = q.u, n = q.n, then = q.then;
        const bool greedy = !(t > 0.0f);
        const double scale = greedy ? 1.0 : scale_of(t);
        __syncthreads();  // (the roots, which every wavefront's look for the part takes; and the state is read before it changes)
        // A listed sequence's state changes in a launch, by the last of its workgroups, after all of them have read it: the first n_seq
        // workgroups leave those alone, whatever they have read. (What is drawn from p behind a draft that fell is drawn there.)
        if (of_p ? q.listed || then != kNone : then == kNone) continue;
        if (n <= 0 || n > a.max_path) continue;
        if (u < 0 || u >= w.n || w.r0 < 0 || w.r0 > a.n_rows - w.n) return;
        for (bool alone = false;;) {
            PartSums early{0.0, 0.0, -INFINITY, -INFINITY, 0, 0};
            if (then == kNone && lane < a.parts) early = a.sums[(int64_t) (w.r0 + u) * a.parts + lane];
            const RowState st = shared(a.state + w.r0 + u);
            const Source z = source(a, w, s, u, st, m.roots, scale);
            if (then == kLeft || then <= kFell) {
#pragma unroll 1
                for (int b = alone ? 0 : own; b < (alone ? a.blocks : own + 1); b++) {
                    const double v = runs(a, z, m, b, false);
                    if (tid < 4 * a.block_steps) agent_store(a.drawn_runs + ((int64_t) s * a.blocks + b) * (4 * a.block_steps) + tid, m.seg[tid]);
                    if (tid == 0) share(a.drawn + (int64_t) s * a.blocks + b, v);
                }
                if (alone) {
                    if (tid == 0) stores_done();
                    __syncthreads();
                } else if (!last_of(&a.seq[s].arrived, a.blocks, &m.flag)) break;
            }
            if (then <= kFell) {
                if (wave == 0) {
                    double C = st.C, c = 0.0;
                    for (int i0 = 0; i0 < a.blocks; i0 += 64) c += wave_sum_d(part_sum(a, z, i0, false, early));
                    const int from = kFell - then;
                    Path on{n, u, decide(a, w, u, from, -1, c, z.p, z.q, children(a, w, u, from + 1), from + 1, C), true, 0};
                    if (tid == 0) {
                        agent_store(&a.state[w.r0 + u].C, C);
                        agent_store(&a.next[w.r0 + u], on.then);
                        stores_done();
                    }
                    if (on.then >= 0 && n < a.max_path) on = follow<true>(a, w, s, n, on.then, 0);
                    if (tid == 0) {
                        path = on;
                        a.count[s] = on.n;
                        a.seq[s].u = on.u, a.seq[s].n = on.then >= 0 ? 0 : on.n, a.seq[s].then = on.then, a.seq[s].arrived = 0;
                        if (on.then >= 0 && on.then < w.n) a.out[(int64_t) s * a.max_path + on.n - 1] = a.tokens[w.r0 + on.then];  // (cut short)
                    }
                }
                __syncthreads();
                u = path.u, n = path.n, then = path.then;
                if (then >= 0 || (then != kNone && !a.last)) break;
                alone = true;
                __syncthreads();
                continue;
            }
            int token = -1;
            if (st.m_p > -INFINITY) {
                token = greedy ? st.top : draw(a, z, m, false, early);
                if (token < 0) {  // (nothing is left, by rounding)
                    RowState all = st;
                    all.C = 0.0;
                    if (lane < a.parts) early = a.sums[(int64_t) (w.r0 + u) * a.parts + lane];
                    token = draw(a, source(a, w, s, u, all, m.roots, scale), m, true, early);
                }
            }
            if (tid == 0) a.out[(int64_t) s * a.max_path + n - 1] = token, a.seq[s].n = 0;
            break;
        }
        __syncthreads();
    }
}

// How a call is cut, and its workspace.
struct VerifyShape {
    int steps, parts;
    int blocks, block_steps;
    size_t items, state, next, arrived, sums, seq, list, drawn, drawn_runs, total;  // offsets
};
VerifyShape verify_shape(int n_seq, int64_t n_rows, int64_t V) {
    VerifyShape z{};
    const auto parts = [&](int steps) { return (V + steps * kStep - 1) / (steps * kStep); };
    // A part costs its steps and some four more; workgroups take theirs in as many turns. Of up to 8 steps: decisions come early enough to
    // spare rows (128256 tokens, 205 rows in 64 chains: 91 us, 92 with up to 16; 800 rows in 16 trees: 66 and 83). Of up to 6 where sequences
    // have many rows, most of which no path comes to (those trees 59, with 4 62). With 6 and with 8: drawn trees, 32 of 18 to 24 rows 138 us and 151, 16
    // of 24 to 32 114 and 118, 16 of 38 to 50 161 and 176; guesses 73 and 75, 57 and 59, 61 and 62, but 64 of 38 to 50 rows 104 and 101. Below 16 rows a
    // sequence: 128 chains of 6 to 8 rows 240 and 244, over 32000 tokens 107 and 96; 64 trees of 6 to 8 rows over those 43 and 40; drawn ones of 12 to 16 188 and 183.
    int64_t best = INT64_MAX;
    for (int k = 2; k <= (n_rows >= 16 * (int64_t) n_seq ? 6 : kSteps); k += 2) {
        const int64_t cost = (n_rows * parts(k) + kRowGroups - 1) / kRowGroups * (k + 4);
        if (cost < best) best = cost, z.steps = k;
    }
    z.parts = (int) parts(z.steps);
    z.items = 256;
    z.state = z.items + align256((size_t) n_rows * sizeof(Item));
    z.next = z.state + align256((size_t) n_rows * sizeof(RowState));
    z.arrived = z.next + align256((size_t) n_rows * sizeof(int));
    z.sums = z.arrived + align256((size_t) n_rows * kApart * sizeof(int));
    z.seq = z.sums + align256((size_t) n_rows * z.parts * sizeof(PartSums));
    z.block_steps = 2;  // (half of the sequences may have something left)
    while (z.block_steps < kSteps && n_seq * parts(z.block_steps) > 2 * kRowGroups) z.block_steps *= 2;
    z.blocks = (int) parts(z.block_steps);
    z.list = z.seq + align256((size_t) n_seq * sizeof(SeqState));
    z.drawn = z.list + align256((size_t) n_seq * sizeof(int));
    z.drawn_runs = z.drawn + align256((size_t) n_seq * z.blocks * sizeof(double));
    z.total = z.drawn_runs + align256((size_t) n_seq * z.blocks * 4 * z.block_steps * sizeof(double));
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

// A wavefront moves one sequence's tokens of one KV head in one cache: a lane has the same code bytes of every token. Eight tokens are read, then
// written, in order: an entry's source is not below its own number, so no earlier target, and nothing is written before it is read.
// Latency (entries, page entries, bytes: 3.3 us), then the lines that it touches, some ten of 128 bytes for the 144 of a token and KV head of
// 128: 32 sequences' paths of up to 7 rows in 32 layers of 8 KV heads 8.2 us; a token at a time 10.
template <int D>
__global__ __launch_bounds__(256) void k_paged_move(const MoveArgs a) {
    constexpr int B = D / 128 > 0 ? D / 128 : 1, N = 8;
    const int lane = threadIdx.x & 63, unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = unit / a.p.Hkv, hk = unit % a.p.Hkv;
    if (s >= a.p.n_seq) return;
    Paged p = a.p;
    p.data = a.data[blockIdx.y];
    const int n = min(a.count[s], a.max_keep);
    const int64_t past = a.p.past[s];
    for (int i0 = 0; i0 < n; i0 += N) {
        // lanes 0 .. 7 look up the sources, 8 .. 15 the targets
        const int e = i0 + (lane & (N - 1)), j = e < n ? a.rows[s * a.ld + e] : -1;
        const int64_t at = lane < 2 * N && j > e ? paged_tile(p, s, past + (lane < N ? j : e), hk, D) : -1;
        const int lo = (int) (uint32_t) at, hi = (int) (at >> 32);
        const auto of = [&](int l) {
            return (int64_t) ((uint64_t) (uint32_t) __builtin_amdgcn_readlane(hi, l) << 32 | (uint32_t) __builtin_amdgcn_readlane(lo, l));
        };
        uint8_t k[N][B], v[N][B];
        uint16_t d[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int64_t src = of(i);
            const int t = (int) (past + __builtin_amdgcn_readlane(j, i)) & 31;
            if (src < 0) continue;
#pragma unroll
            for (int b = 0; b < B; b++)
                if (lane + 64 * b < D / 2) {
                    k[i][b] = p.data[src + paged_k_byte<D>(t, lane + 64 * b)];
                    v[i][b] = p.data[src + paged_v_byte<D>(t, lane + 64 * b)];
                }
            // scales: of K, then of V, which lie as if they were further blocks
            if (lane < D / 16) d[i] = *reinterpret_cast<const uint16_t *>(p.data + src + paged_k_scale<D>(t, lane));
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int64_t src = of(i), dst = of(N + i);
            const int t = (int) (past + i0 + i) & 31;
            if (src < 0 || dst < 0) continue;
#pragma unroll
            for (int b = 0; b < B; b++)
                if (lane + 64 * b < D / 2) {
                    p.data[dst + paged_k_byte<D>(t, lane + 64 * b)] = k[i][b];
                    p.data[dst + paged_v_byte<D>(t, lane + 64 * b)] = v[i][b];
                }
            if (lane < D / 16) *reinterpret_cast<uint16_t *>(p.data + dst + paged_k_scale<D>(t, lane)) = d[i];
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
    const VerifyShape z = verify_shape(n_seq, n_rows, V);
    paged_require((int64_t) n_seq * z.blocks < (1 << 30) && n_rows * z.parts < ((int64_t) 1 << 40), "draft_verify: too many sequences and tokens");
    return z.total;
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
        a.parts = z.parts, a.steps = z.steps;
        a.vec = aligned(logits, 16) && ld % 4 == 0 && (!draft_logits || (aligned(draft_logits, 16) && draft_ld % 4 == 0));
        a.count = count, a.rows = rows, a.out = tokens_out;
        a.n_items = (int *) at, a.n_list = a.n_items + 1, a.items = (Item *) (at + z.items), a.state = (RowState *) (at + z.state);
        a.next = (int *) (at + z.next), a.arrived = (int *) (at + z.arrived), a.sums = (PartSums *) (at + z.sums), a.seq = (SeqState *) (at + z.seq);
        a.list = (int *) (at + z.list), a.drawn = (double *) (at + z.drawn), a.drawn_runs = (double *) (at + z.drawn_runs);
        hipStream_t st = as_stream(stream);
        // (what cannot be launched is refused before the first one)
        const unsigned begin_groups = paged_grid(std::max<int64_t>((n_rows + 3) / 4, 1), kT);
        const unsigned draw_groups = n_rows == 0 ? 0 : paged_grid(n_seq + (draft_logits ? std::min<int64_t>((int64_t) n_seq * z.blocks, 2 * kRowGroups) : 0), kDrawT);
        k_verify_begin<<<begin_groups, kT, 0, st>>>(a);
        check_launch("draft verify");
        if (n_rows == 0) return;
        a.blocks = z.blocks, a.block_steps = z.block_steps;
        a.abreast = (int) std::min<int64_t>(n_rows, std::max(1, kRowGroups / z.parts));
        k_verify_rows<<<paged_grid((int64_t) a.abreast * z.parts, kT + 64), kT + 64, 0, st>>>(a);
        check_launch("draft verify rows");
        // A path that cannot be all of a sequence's rows tells that rows have several drawn children, of which some will fall: a sum of what is left for
        // each, over the chip as often as most need, by one workgroup from there on. (128256 tokens, trees of 20 to 32 rows, one, 4 and 16
        // sequences: 32, 51 and 123 us with three launches, 34, 55 and 100 with five.)
        const int draws = draft_logits && max_path < a.max_rows && z.blocks > 8 ? (n_seq < 8 ? 3 : 5) : 1;
        for (int i = 0; i < draws; i++) {
            a.last = i == draws - 1;
            k_verify_draw<<<draw_groups, kDrawT, 0, st>>>(a);
            check_launch("draft verify draw");
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
            paged_view(caches[c0], batch, 1, false);
            paged_need(caches[c0]->data, "cache data", 16);
            paged_require(caches[c0]->n_pages == caches[0]->n_pages && caches[c0]->page_size == caches[0]->page_size &&
                              caches[c0]->n_head_kv == caches[0]->n_head_kv && caches[c0]->head_dim == caches[0]->head_dim,
                          "paged_move: the caches must be of one shape");
        }
        const size_t size = gcq_paged_cache_size(caches[0]->n_pages, caches[0]->page_size, caches[0]->n_head_kv, caches[0]->head_dim);
        std::vector<uintptr_t> at(n_caches);
        std::transform(caches, caches + n_caches, at.begin(), [](const gcq_paged_cache * c) { return (uintptr_t) c->data; });
        std::sort(at.begin(), at.end());
        for (int i = 1; i < n_caches; i++) paged_require(at[i] - at[i - 1] >= size, "paged_move: caches overlap (a row would move twice)");
        paged_need(batch->pages, "pages", 4);
        paged_need(batch->past, "past", 4);
        if (max_keep == 0) return;
        MoveArgs a{};
        a.p = paged_view(caches[0], batch, 1, false);  // (no starts)
        a.count = count, a.rows = rows, a.ld = ld_rows, a.max_keep = max_keep;
        for (int c0 = 0; c0 < n_caches; c0 += kCaches) {
            const int n = std::min(n_caches - c0, kCaches);
            for (int i = 0; i < n; i++) a.data[i] = (uint8_t *) caches[c0 + i]->data;
            const int64_t x = ((int64_t) batch->n_seq * a.p.Hkv + 3) / 4;
            paged_grid(x * n, 256);
            with_head_dim(caches[0]->head_dim, [&](auto d) { k_paged_move<decltype(d)::value><<<dim3((unsigned) x, n), 256, 0, as_stream(stream)>>>(a); });
            check_launch("paged move");
        }
    });
}

}  // extern "C"
