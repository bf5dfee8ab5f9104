// Verification of drafted tokens against the target's probabilities.
//
// For a sequence with drafted tokens x_0 .. x_{n-1}, target probabilities p_i
// after i of them (i <= n), draft probabilities q_i that x_i was drawn from, and
// uniform numbers u: x_i stands while u_i q_i(x_i) < p_i(x_i); after a of them
// the next token is drawn by the weights
//   w_v = max(p_a(v) - q_a(v), 0)  (a < n),   w_v = p_n(v)  (all stand),
// as the first v at which their running sum exceeds u_K times the whole.  Tokens
// so chosen are distributed as the target's own.
//
// Bound: one row of p and q per sequence, read once for chunks' sums and, of the
// chunk that the token lies in, once more.  Products and sums are in 64 bits:
// what decides is a comparison, and differences of probabilities are small.  64
// sequences, 128000 tokens in fp32: 17 us, the sums 12 (66 MB), the choice 5, a chain
// of latencies; one sequence, 32000 tokens, in one launch: 8.8.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "fkv_paged.h"

namespace fkv {

constexpr int kDraftThreads = 256;
constexpr int kMaxDrafts = 63;      // a lane each, and one for the end
constexpr int kChunkGroups = 4;     // groups of 256 tokens a wave has of a chunk
constexpr int64_t kChunk = 256 * kChunkGroups * (kDraftThreads / 64);  // tokens of a chunk (4096), or a multiple of it
constexpr int kMaxChunks = 512;
constexpr int kSmallGroups = 8;     // ... and of a small vocabulary
constexpr int64_t kSmall = 256 * kSmallGroups * 16;

struct DraftArgs {
    const char* target;
    const char* draft;
    int64_t t_sb, t_sk, d_sb, d_sk;
    const void* tokens;
    const float* uniforms;
    const int32_t* n_draft;
    void* out;
    int32_t* accepted;
    double2* sums;  // workspace: (B, chunks) sums of w and of p
    int32_t K, V, chunk, chunks, is64;
};

template <int DT>
__device__ inline float prob(const char* row, int64_t v) {
    if (DT == FKV_F32) return ((const float*)row)[v];
    const uint16_t w = ((const uint16_t*)row)[v];
    return DT == FKV_F16 ? h2f(w) : bf2f(w);
}

__device__ inline int64_t drafted(const DraftArgs& a, int b, int i) {
    const int64_t at = (int64_t)b * a.K + i;
    return a.is64 ? ((const int64_t*)a.tokens)[at] : (int64_t)((const int32_t*)a.tokens)[at];
}

__device__ inline int drafts_of(const DraftArgs& a, int b) {
    return a.n_draft ? min(max(a.n_draft[b], 0), a.K) : a.K;
}

// The number of the lane below (0 in the first).
__device__ inline double lane_before(double v) { return dpp_or_0<0x138>(v); }  // wave_shr:1

// How many drafted tokens stand (by every wave for itself, a lane a token), and
// of how many.
template <int DT>
__device__ inline int standing(const DraftArgs& a, int b, int& n) {
    const int lane = threadIdx.x & 63;
    n = drafts_of(a, b);
    bool stands = false;
    if (lane < n) {
        const int64_t x = drafted(a, b, lane);
        if (x >= 0 && x < a.V) {  // (a token outside the vocabulary has probability 0)
            const double p = prob<DT>(a.target + b * a.t_sb + lane * a.t_sk, x);
            const double q = a.draft ? (double)prob<DT>(a.draft + b * a.d_sb + lane * a.d_sk, x) : 1.0;
            stands = (double)a.uniforms[(int64_t)b * (a.K + 1) + lane] * q < p;
        }
    }
    return __builtin_ctzll(~__ballot(stands));  // (lane 63 never stands)
}

// Weights of one row.
template <int DT>
struct Weights {
    const char* p;
    const char* q;   // NULL: none to take off,
    int64_t x;       // or all of token x (-1: of none)
    __device__ Weights(const DraftArgs& a, int b, int at, bool rejected) {
        p = a.target + b * a.t_sb + at * a.t_sk;
        q = rejected && a.draft ? a.draft + b * a.d_sb + at * a.d_sk : nullptr;
        x = rejected && !a.draft ? drafted(a, b, at) : -1;
    }
    // (a difference that is not positive, or not a number, has weight 0)
    __device__ double of(float pv, float qv, int64_t v) const {
        const double d = q ? (double)pv - (double)qv : v == x ? 0.0 : (double)pv;
        return d > 0.0 ? d : 0.0;
    }
};

// A block's tokens: wave w has kGroups groups of 256 neighbouring ones from
// first + 256 kGroups w on, four neighbouring ones a lane.
template <int DT, bool VEC, int GROUPS>
__device__ inline void load_weights(const Weights<DT>& w, int64_t first, int64_t last, bool plain, double (&x)[GROUPS][4],
                                    double& whole) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    typedef float f4 __attribute__((ext_vector_type(4)));
    f4 p[GROUPS], q[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const int64_t v = first + 256 * (GROUPS * wave + g) + 4 * lane;
        p[g] = q[g] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        auto four = [&](const char* row) {
            f4 r = {0.0f, 0.0f, 0.0f, 0.0f};
            if (VEC) {  // (rows of a multiple of four tokens, aligned)
                if (v < last) {
                    if (DT == FKV_F32) {
                        r = *(const f4*)(row + 4 * v);
                    } else {
                        const fkv_u2 u = *(const fkv_u2*)(row + 2 * v);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint16_t k = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
                            r[i] = DT == FKV_F16 ? h2f(k) : bf2f(k);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (v + i < last) r[i] = prob<DT>(row, v + i);
            }
            return r;
        };
        p[g] = four(w.p);
        if (w.q) q[g] = four(w.q);
    }
    whole = 0.0;
#pragma unroll
    for (int g = 0; g < GROUPS; g++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double own = p[g][i] > 0.0f ? (double)p[g][i] : 0.0;
            whole += own;
            x[g][i] = plain ? own : w.of(p[g][i], q[g][i], first + 256 * (GROUPS * wave + g) + 4 * lane + i);
        }
}

__device__ inline double of_lane(double v, int i) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), i) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)u, i));
}
__device__ inline double wave_total(double v) {
    v = row_sum(v);
    return (of_lane(v, 0) + of_lane(v, 16)) + (of_lane(v, 32) + of_lane(v, 48));
}
template <int GROUPS>
__device__ inline double lane_total(const double (&x)[GROUPS][4]) {
    double v = 0.0;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) v += (x[g][0] + x[g][1]) + (x[g][2] + x[g][3]);
    return v;
}

// Sums over a block of NT threads, of every thread's two numbers; `sums` keeps the
// waves' of the first.
template <int NT>
__device__ inline void block_sums(double a, double b, double (&sums)[NT / 64], double (&other)[NT / 64], double& sa, double& sb) {
    a = wave_total(a), b = wave_total(b);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = a, other[threadIdx.x >> 6] = b;
    __syncthreads();
    sa = sb = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) sa += sums[w], sb += other[w];
}

// The first token of the block at which the running sum, from `base` on, exceeds
// goal, or the last one with a weight where rounding leaves none; by the waves'
// sums, then a group's, then a lane's.  One thread writes it to *found.
template <int NT, int GROUPS>
__device__ inline void find_token(const double (&x)[GROUPS][4], const double (&sums)[NT / 64], double base, double goal,
                                  int64_t first, int64_t* found) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int chosen = 0;
    double run = base, at = base;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        if (sums[w] > 0.0 && !(at > goal)) chosen = w, run = at;
        at += sums[w];
    }
    if (wave != chosen) return;
    int group = 0;
    double in_group = run;
    at = run;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        const double total = wave_total((x[g][0] + x[g][1]) + (x[g][2] + x[g][3]));
        if (total > 0.0 && !(at > goal)) group = g, in_group = at;
        at += total;
    }
    double y[4] = {};
#pragma unroll
    for (int g = 0; g < GROUPS; g++)
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = group == g ? x[g][i] : y[i];
    const double mine = (y[0] + y[1]) + (y[2] + y[3]);
    double sum = in_group + lane_before(sum_up_to(mine));
    int past = 4, real = -1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        sum += y[i];
        if (y[i] > 0.0) {
            real = i;
            if (past == 4 && sum > goal) past = i;
        }
    }
    const uint64_t hit = __ballot(past < 4), any = __ballot(real >= 0);
    const int64_t v = first + 256 * (GROUPS * wave + group) + 4 * lane;
    if (hit ? lane == __builtin_ctzll(hit) : lane == 63 - __builtin_clzll(any | 1)) *found = v + (hit ? past : max(real, 0));
}

__device__ inline void write_tokens(const DraftArgs& a, int b, int at, int64_t token) {
    const int tid = threadIdx.x;
    if (tid <= a.K) {
        const int64_t x = tid < at ? drafted(a, b, tid) : tid == at ? token : -1;
        const int64_t o = (int64_t)b * (a.K + 1) + tid;
        if (a.is64) ((int64_t*)a.out)[o] = x;
        else ((int32_t*)a.out)[o] = (int32_t)x;
    }
    if (tid == 0) a.accepted[b] = at;
}

// Sums of one chunk.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kDraftThreads) draft_sums_kernel(DraftArgs a) {
    __shared__ double sums[kDraftThreads / 64], other[kDraftThreads / 64];
    const int b = blockIdx.y;
    int n;
    const int at = standing<DT>(a, b, n);
    const Weights<DT> w(a, b, at, at < n);
    const int64_t first = (int64_t)blockIdx.x * a.chunk, last = min(first + a.chunk, (int64_t)a.V);
    double sum = 0.0, whole = 0.0;
    for (int64_t v = first; v < last; v += kChunk) {
        double x[kChunkGroups][4], y;
        load_weights<DT, VEC, kChunkGroups>(w, v, last, false, x, y);
        sum += lane_total(x);
        whole += y;
    }
    block_sums<kDraftThreads>(sum, whole, sums, other, sum, whole);
    if (threadIdx.x == 0) {
        a.sums[(int64_t)b * a.chunks + blockIdx.x] = make_double2(sum, whole);
        if (blockIdx.x == 0) a.accepted[b] = at;
    }
}

// The next token of one sequence from its chunks' sums, 64 a step, and its results.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kDraftThreads) draft_choice_kernel(DraftArgs a) {
    constexpr int S = kMaxChunks / 64;
    __shared__ double sums[kDraftThreads / 64], other[kDraftThreads / 64];
    __shared__ int64_t found;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    double2 of[S];
#pragma unroll
    for (int j = 0; j < S; j++) {
        const int i = 64 * j + lane;
        of[j] = i < a.chunks ? a.sums[(int64_t)b * a.chunks + i] : make_double2(0.0, 0.0);
    }
    const int at = a.accepted[b];  // (draft_sums_kernel's)
    const Weights<DT> w(a, b, at, at < drafts_of(a, b));
    if (tid == 0) found = -1;
    __syncthreads();
    double total = 0.0, whole = 0.0;
#pragma unroll
    for (int j = 0; j < S; j++)
        if (64 * j < a.chunks) total += wave_total(of[j].x), whole += wave_total(of[j].y);
    // Nothing left of the target's row (p <= q everywhere, by rounding): its own
    // probabilities.
    const bool plain = !(total > 0.0);
    if (plain) total = whole;
    if (total > 0.0 && total < (double)INFINITY) {
        const double goal = (double)a.uniforms[(int64_t)b * (a.K + 1) + a.K] * total;
        // the chunk in which the running sum passes it: the last one with a weight that it
        // reaches before
        double sum = 0.0, base = 0.0;
        int c = 0;
#pragma unroll
        for (int j = 0; j < S; j++)
            if (64 * j < a.chunks) {
                const double own = plain ? of[j].y : of[j].x, upto = sum_up_to(own), before = sum + lane_before(upto);
                const uint64_t reached = __ballot(own > 0.0 && !(before > goal));
                if (reached) {
                    const int i = 63 - __builtin_clzll(reached);
                    c = 64 * j + i, base = of_lane(before, i);
                }
                sum += of_lane(upto, 63);
            }
        const int64_t first = (int64_t)c * a.chunk, last = min(first + a.chunk, (int64_t)a.V);
        // (a chunk of several blocks, by a vocabulary of more than 2^21: one by one)
        for (int64_t v = first; v < last; v += kChunk) {
            double x[kChunkGroups][4], y, block;
            load_weights<DT, VEC, kChunkGroups>(w, v, last, plain, x, y);
            block_sums<kDraftThreads>(lane_total(x), 0.0, sums, other, block, y);
            if (block > 0.0) find_token<kDraftThreads>(x, sums, base, goal, v, &found);
            base += block;
            __syncthreads();
            if (base > goal) break;
        }
    }
    __syncthreads();
    write_tokens(a, b, at, found);
}

// Both in one for a small vocabulary, a workgroup a sequence: one launch, and each
// probability read once.
template <int DT, bool VEC>
__global__ void __launch_bounds__(1024) draft_small_kernel(DraftArgs a) {
    __shared__ double sums[16], other[16];
    __shared__ int64_t found;
    const int b = blockIdx.x;
    if (threadIdx.x == 0) found = -1;
    int n;
    const int at = standing<DT>(a, b, n);
    const Weights<DT> w(a, b, at, at < n);
    double x[kSmallGroups][4], whole, total;
    load_weights<DT, VEC, kSmallGroups>(w, 0, a.V, false, x, whole);
    block_sums<1024>(lane_total(x), whole, sums, other, total, whole);
    const bool plain = !(total > 0.0);
    if (plain) {  // (the same for the whole workgroup)
        __syncthreads();
        load_weights<DT, VEC, kSmallGroups>(w, 0, a.V, true, x, whole);
        block_sums<1024>(lane_total(x), 0.0, sums, other, total, whole);
    }
    if (total > 0.0 && total < (double)INFINITY)
        find_token<1024>(x, sums, 0.0, (double)a.uniforms[(int64_t)b * (a.K + 1) + a.K] * total, 0, &found);
    __syncthreads();
    write_tokens(a, b, at, found);
}

struct DraftPlan {
    int64_t chunk, chunks;
};
static DraftPlan plan_drafts(int32_t V) {
    DraftPlan r;
    r.chunk = std::max<int64_t>(kChunk, round_up(cdiv(V, kMaxChunks), kChunk));
    r.chunks = cdiv(V, r.chunk);
    return r;
}
static int check_drafts(const char* who, int32_t B, int32_t K, int32_t V) {
    const std::string w = who;
    if (B < 0 || B > 65535) return set_error(w + ": at most 65535 sequences");
    if (K < 0 || K > kMaxDrafts) return set_error(w + ": at most 63 drafted tokens");
    if (V < 1) return set_error(w + ": the vocabulary is empty");
    return FKV_OK;
}

}  // namespace fkv

using namespace fkv;

extern "C" {

int64_t fkv_verify_drafts_workspace(int32_t B, int32_t K, int32_t V) {
    if (int e = check_drafts("fkv_verify_drafts_workspace", B, K, V)) return e;
    return 16 * B * plan_drafts(V).chunks;
}

int fkv_verify_drafts(const fkv_rows* target, const fkv_rows* draft, int32_t dtype, int32_t B, int32_t K, int32_t V,
                      const void* tokens, int32_t tokens64, const float* uniforms, const int32_t* n_draft,
                      void* out_tokens, int32_t* accepted, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* w = "fkv_verify_drafts";
    if (int e = check_drafts(w, B, K, V)) return e;
    if (dtype < FKV_F16 || dtype > FKV_F32) return set_error(std::string(w) + ": unknown dtype");
    if (B == 0) return FKV_OK;
    if (!target || !target->data || (draft && !draft->data && K > 0) || (K > 0 && !tokens) || !uniforms || !out_tokens || !accepted)
        return set_error(std::string(w) + ": NULL argument");
    const DraftPlan p = plan_drafts(V);
    if (!workspace || (uintptr_t)workspace & 15 || workspace_bytes < 16 * B * p.chunks)
        return set_error(std::string(w) + ": 16-byte aligned workspace of " + std::to_string(16 * B * p.chunks) + " bytes needed");
    const int64_t es = dtype == FKV_F32 ? 4 : 2;
    DraftArgs a;
    a.target = (const char*)target->data;
    a.t_sb = target->stride_b * es;
    a.t_sk = target->stride_l * es;
    a.draft = draft && K > 0 ? (const char*)draft->data : nullptr;
    a.d_sb = draft ? draft->stride_b * es : 0;
    a.d_sk = draft ? draft->stride_l * es : 0;
    a.tokens = tokens;
    a.uniforms = uniforms;
    a.n_draft = n_draft;
    a.out = out_tokens;
    a.accepted = accepted;
    a.sums = (double2*)workspace;
    a.K = K;
    a.V = V;
    a.chunk = (int32_t)p.chunk;
    a.chunks = (int32_t)p.chunks;
    a.is64 = tokens64 != 0;
    // (four tokens a load, which rows of a multiple of four allow)
    const bool vec = !(((uintptr_t)a.target | a.t_sb | a.t_sk | (uintptr_t)a.draft | a.d_sb | a.d_sk | V * es) & (4 * es - 1));
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (V <= kSmall)
            return start_kernel(w, vec ? draft_small_kernel<DT, true> : draft_small_kernel<DT, false>, B, 1024, s, a);
        const dim3 grid((uint32_t)p.chunks, B);
        if (int e = start_kernel(w, vec ? draft_sums_kernel<DT, true> : draft_sums_kernel<DT, false>, grid, kDraftThreads, s, a))
            return e;
        return start_kernel(w, vec ? draft_choice_kernel<DT, true> : draft_choice_kernel<DT, false>, B, kDraftThreads, s, a);
    };
    if (dtype == FKV_F16) return go(std::integral_constant<int, FKV_F16>{});
    if (dtype == FKV_BF16) return go(std::integral_constant<int, FKV_BF16>{});
    return go(std::integral_constant<int, FKV_F32>{});
}

}  // extern "C"
