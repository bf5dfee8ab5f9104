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
// what decides is a comparison, and differences of probabilities are small.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "fkv_paged.h"

namespace fkv {

constexpr int kDraftThreads = 256;
constexpr int kMaxDrafts = 63;      // a lane each, and one for the end
constexpr int64_t kChunk = 4096;    // tokens of a vocabulary's chunk, or more
constexpr int kMaxChunks = 512;

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

// How many drafted tokens stand (by every wave for itself, a lane a token), and
// of how many.
template <int DT>
__device__ inline int standing(const DraftArgs& a, int b, int& n) {
    const int lane = threadIdx.x & 63;
    n = a.n_draft ? min(max(a.n_draft[b], 0), a.K) : a.K;
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
    __device__ double at(int64_t v) const { return of(prob<DT>(p, v), q ? prob<DT>(q, v) : 0.0f, v); }
    __device__ double plain(int64_t v) const {
        const double d = prob<DT>(p, v);
        return d > 0.0 ? d : 0.0;
    }
};

__device__ inline double block_sum(double v, double* lds) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += wave_xor(v, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kDraftThreads / 64; w++) v += lds[w];
    __syncthreads();
    return v;
}

// Sums of one chunk.  VEC: rows are 16-byte aligned and of a multiple of 16 bytes.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kDraftThreads) draft_sums_kernel(DraftArgs a) {
    __shared__ double lds[kDraftThreads / 64];
    const int b = blockIdx.y;
    int n;
    const int at = standing<DT>(a, b, n);
    const Weights<DT> w(a, b, at, at < n);
    const int64_t first = (int64_t)blockIdx.x * a.chunk, last = min(first + a.chunk, (int64_t)a.V);
    double sum = 0.0, whole = 0.0;
    if (VEC) {
        constexpr int N = DT == FKV_F32 ? 4 : 8;  // of a load
        constexpr int U = 4;
        const fkv_u4 none = {0, 0, 0, 0};
        for (int64_t v0 = first + N * threadIdx.x; v0 < last; v0 += U * N * kDraftThreads) {
            fkv_u4 x[U], y[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int64_t v = v0 + u * N * kDraftThreads;
                const bool in = v < last;
                x[u] = in ? *(const fkv_u4*)(w.p + v * (16 / N)) : none;
                y[u] = in && w.q ? *(const fkv_u4*)(w.q + v * (16 / N)) : none;
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < N; i++) {
                    auto value = [&](const fkv_u4& r) {
                        if (DT == FKV_F32) return __uint_as_float(r[i % 4]);
                        const uint16_t k = (uint16_t)(r[i / 2 % 4] >> (16 * (i & 1)));
                        return DT == FKV_F16 ? h2f(k) : bf2f(k);
                    };
                    const float p = value(x[u]);
                    sum += w.of(p, value(y[u]), v0 + u * N * kDraftThreads + i);
                    whole += p > 0.0f ? (double)p : 0.0;
                }
        }
    } else {
        for (int64_t v = first + threadIdx.x; v < last; v += kDraftThreads) {
            sum += w.at(v);
            whole += w.plain(v);
        }
    }
    sum = block_sum(sum, lds);
    whole = block_sum(whole, lds);
    if (threadIdx.x == 0) a.sums[(int64_t)b * a.chunks + blockIdx.x] = make_double2(sum, whole);
}

// The next token of one sequence, and its results.
template <int DT>
__global__ void __launch_bounds__(kDraftThreads) draft_choice_kernel(DraftArgs a) {
    __shared__ double chunk_sum[2][kMaxChunks], before[kDraftThreads / 64];
    __shared__ int64_t found, last_real;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int n;
    const int at = standing<DT>(a, b, n);
    const Weights<DT> w(a, b, at, at < n);
    for (int i = tid; i < a.chunks; i += kDraftThreads) {
        const double2 s = a.sums[(int64_t)b * a.chunks + i];
        chunk_sum[0][i] = s.x, chunk_sum[1][i] = s.y;
    }
    if (tid == 0) found = last_real = -1;
    __syncthreads();
    double total = 0.0, whole = 0.0;
    for (int i = 0; i < a.chunks; i++) total += chunk_sum[0][i], whole += chunk_sum[1][i];
    // Nothing left of the target's row (p <= q everywhere, by rounding): its own
    // probabilities.
    const bool plain = !(total > 0.0);
    if (plain) total = whole;
    int64_t token = -1;
    if (total > 0.0 && total < (double)INFINITY) {
        const double goal = (double)a.uniforms[(int64_t)b * (a.K + 1) + a.K] * total;
        // the chunk in which the running sum passes it (rounding: or the last with any weight)
        double sum = 0.0, base = 0.0;
        int c = 0;
        for (int i = 0; i < a.chunks; i++) {
            const double s = chunk_sum[plain][i];
            if (s > 0.0) c = i, base = sum;
            sum += s;
            if (sum > goal) break;
        }
        const int64_t first = (int64_t)c * a.chunk, last = min(first + a.chunk, (int64_t)a.V);
        const int64_t per = (a.chunk + kDraftThreads - 1) / kDraftThreads;
        const int64_t v0 = min(first + tid * per, last), v1 = min(v0 + per, last);
        double mine = 0.0;
        int64_t real = -1;
        for (int64_t v = v0; v < v1; v++) {
            const double x = plain ? w.plain(v) : w.at(v);
            mine += x;
            if (x > 0.0) real = v;
        }
        double sums = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(sums, o, 64);
            if (lane >= o) sums += x;
        }
        if (lane == 63) before[wave] = sums;
        __syncthreads();
        double run = base + (sums - mine);
        for (int i = 0; i < wave; i++) run += before[i];
        // the first token, over all threads, at which the running sum passes it
        int64_t mine_at = -1;
        for (int64_t v = v0; v < v1; v++) {
            const double x = plain ? w.plain(v) : w.at(v);
            run += x;
            if (x > 0.0 && run > goal) {
                mine_at = v;
                break;
            }
        }
        atomicMin((unsigned long long*)&found, (unsigned long long)mine_at);  // (-1: above all)
        atomicMax((long long*)&last_real, (long long)real);
        __syncthreads();
        token = found >= 0 ? found : last_real;
    }
    if (tid <= a.K) {
        const int64_t x = tid < at ? drafted(a, b, tid) : tid == at ? token : -1;
        const int64_t o = (int64_t)b * (a.K + 1) + tid;
        if (a.is64) ((int64_t*)a.out)[o] = x;
        else ((int32_t*)a.out)[o] = (int32_t)x;
    }
    if (tid == 0) a.accepted[b] = at;
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
    const bool vec = !(((uintptr_t)a.target | a.t_sb | a.t_sk | (uintptr_t)a.draft | a.d_sb | a.d_sk | V * es) & 15);
    hipStream_t s = (hipStream_t)stream;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const dim3 grid((uint32_t)p.chunks, B);
        if (int e = start_kernel(w, vec ? draft_sums_kernel<DT, true> : draft_sums_kernel<DT, false>, grid, kDraftThreads, s, a))
            return e;
        return start_kernel(w, draft_choice_kernel<DT>, B, kDraftThreads, s, a);
    };
    if (dtype == FKV_F16) return go(std::integral_constant<int, FKV_F16>{});
    if (dtype == FKV_BF16) return go(std::integral_constant<int, FKV_BF16>{});
    return go(std::integral_constant<int, FKV_F32>{});
}

}  // extern "C"
