// Routing of tokens to experts: softmax over the experts, the k most probable of them with their weights, the rows per expert as
// ascb200_grouped_gemm takes them, a balance loss, and the gradients of both.
//
//   p[t, e] = softmax over the unmasked experts of logits[t]          (a logit of -inf masks its expert)
//   idx[t, j], weights[t, j]: the j-th largest, ties to the lower index; weights p or p / sum of the chosen p
//   counts[e] = tokens that chose e,   N = tokens in use,   P[e] = sum_t p[t, e] / N
//   loss = E / (N top_k) * sum_e counts[e] * P[e]                     (1 for perfect balance)
//
// Gradients (counts are constants): dp[t, e] = dloss * E * counts[e] / (N^2 top_k) + (what the weights' gradient gives the chosen),
// dlogits = p * (dp - sum_e p dp).
//
// One token per warp, its logits in registers (expert e in lane e % 32).  The sums over tokens stay in registers, then shared
// memory, then one row of the workspace per block; a second kernel adds these rows in block order.  Integer atomics only, so
// every output is reproducible.
#include <algorithm>

#include "common.cuh"

namespace ascb200 {
namespace {

constexpr int kMaxExperts = 1024;     // what ascb200_grouped_gemm takes
constexpr int kMaxTopK = 32;          // one choice per lane
constexpr int kRouteWarps = 16;       // tokens at a time per block
// Rows of the workspace, whose size a caller asks for without a device: two blocks on each of a B200's 148 SMs (us with 148 / 296 / 592: 32768 x 256 fp32, 8 choices
// 40 / 27 / 32, 32768 x 64 bf16, 6 choices 27 / 18 / 21, 4096 x 128 bf16, 8 choices 9.1 / 8.6 / 8.6).
constexpr int kMaxRouteBlocks = 296;
constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned kAll = 0xFFFFFFFFu;

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return f32_to_f16_sat(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return f32_to_bf16(v); }

// Largest of a warp's values; NaN only where all are.
__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float kNegInf = -__builtin_huge_valf();

// The choice works on one integer per logit: its bits in their order (as signed integers), with the expert in the low bits, the lower
// expert larger.  The largest integer of the warp is then the next choice and its expert at once, and a lane keeps its three
// largest with five integer minima and maxima per logit.  (Comparing values and carrying expert numbers beside them took 730
// instructions per token of 256 experts and 8 choices, bound by the integer pipe; this takes about half.)  A 16-bit logit has at least 13
// low zero bits as fp32, so this is exact; an fp32 logit loses its low bits to the expert, so a token among whose choices, or behind
// the last of them, two neighbours agree in the remaining bits is chosen again exactly (choose_exactly).
constexpr int kNoChoice = static_cast<int>(0x80000000u);
constexpr int kLowest = static_cast<int>(0x80800000u);  // -FLT_MAX; smaller: -inf, or nothing
__device__ __forceinline__ int order_key(float x, int e, int low_bits)
{
    const int b = __float_as_int(__fadd_rn(x, 0.0f));  // -0 as +0
    return ((b ^ ((b >> 31) & 0x7FFFFFFF)) & ~low_bits) | (low_bits - e);
}
// The logit of a key, exactly where the logit's low bits are zero: those of a negative one are ones in the order.
__device__ __forceinline__ float key_value(int key, int low_bits)
{
    const int b = key < 0 ? key | low_bits : key & ~low_bits;
    return __int_as_float(b ^ ((b >> 31) & 0x7FFFFFFF));
}
struct Best3 {
    int v1, v2, v3, held;
    template <int NV>
    __device__ __forceinline__ void scan(const int (&key)[NV], int below)
    {
        v1 = v2 = v3 = kNoChoice;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = key[i] < below ? key[i] : kNoChoice;
            v3 = max(v3, min(v2, k));
            v2 = max(v2, min(v1, k));
            v1 = max(v1, k);
        }
        held = 3;
    }
    template <int NV>
    __device__ __forceinline__ void scan(const int (&key)[NV])
    {
        v1 = v2 = v3 = kNoChoice;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v3 = max(v3, min(v2, key[i]));
            v2 = max(v2, min(v1, key[i]));
            v1 = max(v1, key[i]);
        }
        held = 3;
    }
};

// Choice number `lane` of a token by comparisons of the values themselves: numbers in descending order, then NaN, equal ones in the order of
// the experts; -inf never.  One pass over a lane's logits per choice: for the rare tokens.
template <typename T, int NV>
__device__ __noinline__ int choose_exactly(const T* row, int E, int K, int lane)
{
    float x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = lane + 32 * i < E ? to_f32(row[lane + 32 * i]) : kNegInf;
    int my_idx = -1;
    float last = __builtin_huge_valf();
    int last_e = -1;
    bool nan = false;  // the numbers are used up
    for (int j = 0; j < K; ++j) {
        float v = kNegInf;
        int e = kMaxExperts;
        if (!nan) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {  // (comparisons with a NaN are false)
                const int f = lane + 32 * i;
                if ((x[i] < last || (x[i] == last && f > last_e)) && x[i] > v) v = x[i], e = f;
            }
            const float top = warp_max(v);
            nan = top == kNegInf;
            if (!nan) {
                e = __reduce_min_sync(kAll, v == top ? e : kMaxExperts);
                last = top;
            } else {
                last_e = -1;
            }
        }
        if (nan) {
            e = kMaxExperts;
#pragma unroll
            for (int i = NV - 1; i >= 0; --i)
                if (x[i] != x[i] && lane + 32 * i > last_e) e = lane + 32 * i;
            e = __reduce_min_sync(kAll, e);
            if (e == kMaxExperts) break;
        }
        if (lane == j) my_idx = e;
        last_e = e;
    }
    return my_idx;
}

struct RouteArgs {
    const void* logits;
    const uint8_t* valid;
    int* idx;
    float* weights;
    long long* counts;
    long long* num_tokens;
    float* prob_mean;
    float* loss;
    float* part_prob;  // [blocks][experts]
    int* part_count;   // [blocks][experts]
    int* part_tokens;  // [blocks]
    long long ld;
    int tokens, experts, top_k, renorm;
};

// loss, means and counts from the sums of one expert; returns the expert's share of sum_e counts[e] P[e].
__device__ __forceinline__ float finish_expert(const RouteArgs& p, int e, float prob, int count, float inv_n)
{
    const float mean = prob * inv_n;
    if (p.counts) p.counts[e] = count;
    if (p.prob_mean) p.prob_mean[e] = mean;
    return static_cast<float>(count) * mean;
}
__device__ __forceinline__ float loss_of(const RouteArgs& p, float total, float inv_n)
{
    return total * inv_n * (static_cast<float>(p.experts) / static_cast<float>(p.top_k));
}

// A block has a run of consecutive tokens, which it takes in tiles of one token per thread: it first writes down which of the tile's tokens
// are valid (and closes the others), then its warps share those evenly.  FULL: the experts are 32 NV exactly.
template <typename T, int NV, bool FULL>
__global__ void __launch_bounds__(kRouteWarps * 32, NV <= 8 ? 2 : 1)
route_kernel(const RouteArgs p)
{
    constexpr int TILE = kRouteWarps * 32;
    constexpr int low_bits = 32 * NV - 1;  // at most 1023; the numbers of all lanes' experts fit
    constexpr bool AHEAD = NV <= 16;       // the next token's logits are requested before this one's are worked on
    extern __shared__ float s_prob[];      // [kRouteWarps][experts], then int [experts] counts
    __shared__ int s_tokens[kRouteWarps];
    __shared__ float s_part[kRouteWarps];
    __shared__ uint16_t s_list[TILE];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int E = FULL ? 32 * NV : p.experts, K = p.top_k;
    int* s_count = reinterpret_cast<int*>(s_prob + kRouteWarps * E);
    for (int e = threadIdx.x; e < E; e += kRouteWarps * 32) s_count[e] = 0;
    grid_dependency_wait();
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
    int used = 0;
    const int run = static_cast<int>((p.tokens + static_cast<long long>(gridDim.x) - 1) / gridDim.x);
    const long long first = static_cast<long long>(blockIdx.x) * run;
    const int mine = static_cast<int>(max(0ll, min(static_cast<long long>(run), p.tokens - first)));
    for (int tile = 0; tile < mine; tile += TILE) {
        const long long token0 = first + tile;
        int count = min(TILE, mine - tile);
        __syncthreads();  // the zeroed counts; the list of the tile before
        if (p.valid) {
            const bool inside = static_cast<int>(threadIdx.x) < count;
            const bool open = inside && p.valid[token0 + threadIdx.x] != 0;
            const unsigned votes = __ballot_sync(kAll, open);
            if (lane == 0) s_tokens[w] = __popc(votes);
            __syncthreads();
            int before = 0, all = 0;
#pragma unroll
            for (int i = 0; i < kRouteWarps; ++i) {
                before += i < w ? s_tokens[i] : 0;
                all += s_tokens[i];
            }
            if (open) {
                s_list[before + __popc(votes & ((1u << lane) - 1))] = static_cast<uint16_t>(threadIdx.x);
            } else if (inside) {
                for (int j = 0; j < K; ++j) {
                    p.idx[(token0 + threadIdx.x) * K + j] = -1;
                    p.weights[(token0 + threadIdx.x) * K + j] = 0.0f;
                }
            }
            count = all;
            __syncthreads();
        }
        const T* rows = static_cast<const T*>(p.logits) + token0 * p.ld + lane;
        const long long ld = p.ld;
        int* idx_out = p.idx + token0 * K + lane;
        float* weights_out = p.weights + token0 * K + lane;
        auto load = [&](int j, const T*& row, T (&to)[NV]) {
            const int t = p.valid ? s_list[min(j, TILE - 1)] : j;
            row = rows + t * ld;
            if (j >= count) return t;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (FULL || lane + 32 * i < E) to[i] = row[32 * i];
            return t;
        };
        T raw[NV], ahead[NV];
        const T *row, *row_ahead;
        int t, t_ahead = 0;
        if constexpr (AHEAD) t_ahead = load(w, row_ahead, ahead);
        for (int j = w; j < count; j += kRouteWarps) {
            if constexpr (AHEAD) {
#pragma unroll
                for (int i = 0; i < NV; ++i) raw[i] = ahead[i];
                row = row_ahead, t = t_ahead;
                t_ahead = load(j + kRouteWarps, row_ahead, ahead);
            } else {
                t = load(j, row, raw);
            }
            float x[NV];
            int key[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                x[i] = FULL || lane + 32 * i < E ? to_f32(raw[i]) : kNegInf;
                key[i] = order_key(x[i], lane + 32 * i, low_bits);
            }
            Best3 best;
            best.scan(key);
            int top = __reduce_max_sync(kAll, best.v1);
            float m;  // the largest logit, exactly: a few low bits of a value beyond 1e6 less would make exp(x - m) overflow
            if constexpr (sizeof(T) == 2) {
                m = key_value(top, low_bits);
            } else {
                m = kNegInf;
#pragma unroll
                for (int i = 0; i < NV; ++i) m = fmaxf(m, x[i]);
                m = warp_max(m);
            }
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                x[i] = exp2_approx((x[i] - m) * kLog2e);
                sum += x[i];
            }
            sum = warp_sum(sum);
            const bool not_a_number = sum != sum;  // a NaN or +inf among the logits, or all of them masked (-inf less -inf)
            int my_key = kNoChoice;
            int chosen = 0;
            for (; chosen < K && top >= kLowest; ++chosen) {
                if (lane == chosen) my_key = top;
                if (best.v1 == top) {
                    best.v1 = best.v2, best.v2 = best.v3, best.v3 = kNoChoice;
                    if (--best.held == 0) best.scan(key, top);  // one token in twenty with 8 choices among 32 lanes
                }
                top = __reduce_max_sync(kAll, best.v1);
            }
            int my_idx = my_key != kNoChoice ? low_bits - (my_key & low_bits) : -1;
            bool again = not_a_number;
            if constexpr (sizeof(T) == 4) {
                const int next = __shfl_down_sync(kAll, my_key, 1);
                const int behind = lane == chosen - 1 ? top : next;  // what was left behind the last choice
                again |= __any_sync(kAll, lane < chosen && ((my_key ^ behind) & ~low_bits) == 0);
            }
            if (again) my_idx = choose_exactly<T, NV>(row - lane, E, K, lane);
            float my_w = 0.0f;
            if (__any_sync(kAll, my_idx >= 0)) {
                ++used;
                const float inv = rcp_approx(sum);
#pragma unroll
                for (int i = 0; i < NV; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
                if (my_idx >= 0) {
                    my_w = exp2_approx((to_f32(row[my_idx - lane]) - m) * kLog2e) * inv;
                    atomicAdd(&s_count[my_idx], 1);
                }
                if (p.renorm) {
                    const float total = warp_sum(my_w);  // lanes without a choice hold 0
                    if (my_idx >= 0) my_w *= rcp_approx(total);
                }
            }
            if (lane < K) {
                idx_out[t * K] = my_idx;  // less than TILE * kMaxTopK
                weights_out[t * K] = my_w;
            }
        }
    }
    __syncthreads();  // every count is in; s_tokens is free again
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (lane + 32 * i < E) s_prob[w * E + lane + 32 * i] = acc[i];
    if (lane == 0) s_tokens[w] = used;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int i = 0; i < kRouteWarps; ++i) n += s_tokens[i];
    const float inv_n = __frcp_rn(static_cast<float>(max(n, 1)));
    float share = 0.0f;
    for (int e = threadIdx.x; e < E; e += kRouteWarps * 32) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < kRouteWarps; ++i) v += s_prob[i * E + e];
        if (gridDim.x == 1) {
            share += finish_expert(p, e, v, s_count[e], inv_n);
        } else {
            p.part_prob[static_cast<size_t>(blockIdx.x) * E + e] = v;
            p.part_count[static_cast<size_t>(blockIdx.x) * E + e] = s_count[e];
        }
    }
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) p.part_tokens[blockIdx.x] = n;
        return;
    }
    share = warp_sum(share);
    if (lane == 0) s_part[w] = share;
    __syncthreads();
    if (threadIdx.x == 0) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kRouteWarps; ++i) total += s_part[i];
        if (p.loss) p.loss[0] = loss_of(p, total, inv_n);
        if (p.num_tokens) p.num_tokens[0] = n;
    }
}

// Adds the blocks' rows.  One cluster of eight blocks; each takes an eighth of the experts, 32 at a time, its 32 warps every 32nd row
// each (ten loads per thread, all in flight); the shares of the loss meet in the first block's shared memory.
constexpr int kFinishBlocks = 8, kFinishWarps = 32;
__global__ void __cluster_dims__(kFinishBlocks, 1, 1) __launch_bounds__(kFinishWarps * 32)
route_finish_kernel(const RouteArgs p, int blocks)
{
    __shared__ float s_p[kFinishWarps][32];
    __shared__ int s_c[kFinishWarps][32];
    __shared__ int s_n[kFinishWarps];
    __shared__ float s_loss[kFinishBlocks];
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for below: every block of the cluster has started
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int n = static_cast<int>(threadIdx.x) < blocks ? p.part_tokens[threadIdx.x] : 0;
    n = __reduce_add_sync(kAll, n);
    if (lane == 0) s_n[w] = n;
    const int per = (p.experts + kFinishBlocks - 1) / kFinishBlocks;
    const int e1 = min(p.experts, (static_cast<int>(blockIdx.x) + 1) * per);
    float share = 0.0f, inv_n = 0.0f;
    int total_n = 0;
    for (int base = blockIdx.x * per; base < (static_cast<int>(blockIdx.x) + 1) * per; base += 32) {
        const int e = base + lane;
        float v = 0.0f;
        int c = 0;
        if (e < e1) {
#pragma unroll 10
            for (int b = w; b < blocks; b += kFinishWarps) {
                v += p.part_prob[static_cast<size_t>(b) * p.experts + e];
                c += p.part_count[static_cast<size_t>(b) * p.experts + e];
            }
        }
        __syncthreads();
        s_p[w][lane] = v, s_c[w][lane] = c;
        __syncthreads();
        if (w == 0) {
            total_n = __reduce_add_sync(kAll, s_n[lane]);
            inv_n = __frcp_rn(static_cast<float>(max(total_n, 1)));
            if (e < e1) {
#pragma unroll
                for (int i = 1; i < kFinishWarps; ++i) v += s_p[i][lane], c += s_c[i][lane];
                share += finish_expert(p, e, v, c, inv_n);
            }
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (w == 0) {
        share = warp_sum(share);
        if (lane == 0) {
            uint32_t slot = static_cast<uint32_t>(__cvta_generic_to_shared(&s_loss[blockIdx.x])), first;
            asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(slot));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(first), "f"(share) : "memory");
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kFinishBlocks; ++i) total += s_loss[i];
        if (p.loss) p.loss[0] = loss_of(p, total, inv_n);
        if (p.num_tokens) p.num_tokens[0] = total_n;
    }
}

struct RouteGradArgs {
    const void* logits;
    const int* idx;
    const long long* counts;
    const long long* num_tokens;
    const float* dloss;
    const float* dweights;
    void* dlogits;
    long long ld, ld_out;
    int tokens, experts, top_k, renorm;
};

// One token per warp.  With E_i = exp(x_i - max) and S their sum: p_i = E_i / S, and sum_e p dp = (sum_i E_i base_i) / S + sum_j p_j g_j with
// base_e = dloss E counts[e] / (N^2 top_k) and g_j what the weights' gradient gives choice j: every sum over experts is made from
// values in registers.  The lanes write p (base - sum) for their experts, and after that the choices' own lanes write theirs again with
// g_j in it.
template <typename T, int NV, bool FULL>
__global__ void __launch_bounds__(256)
route_grad_kernel(const RouteGradArgs p)
{
    extern __shared__ float s_base[];  // [experts]
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int E = FULL ? 32 * NV : p.experts, K = p.top_k;
    grid_dependency_wait();
    float coef = 0.0f;
    if (p.dloss) {
        const float n = static_cast<float>(max(*p.num_tokens, 1ll));
        coef = *p.dloss * static_cast<float>(E) / (n * n * static_cast<float>(K));
    }
    for (int e = threadIdx.x; e < E; e += 256) s_base[e] = p.dloss ? coef * static_cast<float>(p.counts[e]) : 0.0f;
    __syncthreads();
    float base[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) base[i] = FULL || lane + 32 * i < E ? s_base[lane + 32 * i] : 0.0f;
    const long long step = static_cast<long long>(gridDim.x) * 8;
    long long t = static_cast<long long>(blockIdx.x) * 8 + w;
    constexpr bool AHEAD = NV <= 16;  // the next token is requested before this one is worked on
    T raw[NV], raw_ahead[NV];
    int my = -1, my_ahead = -1;
    float gw = 0.0f, gw_ahead = 0.0f;
    auto load = [&](long long token, T (&to)[NV], int& idx, float& g) {
        if (token >= p.tokens) return;
        const T* row = static_cast<const T*>(p.logits) + token * p.ld;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (FULL || lane + 32 * i < E) to[i] = row[lane + 32 * i];
        if (lane < K) {
            idx = p.idx[token * K + lane];
            if (p.dweights) g = p.dweights[token * K + lane];
        }
    };
    if constexpr (AHEAD) load(t, raw_ahead, my_ahead, gw_ahead);
    for (; t < p.tokens; t += step) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < NV; ++i) raw[i] = raw_ahead[i];
            my = my_ahead, gw = gw_ahead;
            load(t + step, raw_ahead, my_ahead, gw_ahead);
        } else {
            load(t, raw, my, gw);
        }
        const T* row = static_cast<const T*>(p.logits) + t * p.ld;
        T* out = static_cast<T*>(p.dlogits) + t * p.ld_out;
        const bool mine = my >= 0 && my < E;
        if (!__any_sync(kAll, mine)) {  // not in use
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (FULL || lane + 32 * i < E) out[lane + 32 * i] = from_f32<T>(0.0f);
            continue;
        }
        const float my_logit = mine ? to_f32(row[my]) : 0.0f;
        __syncwarp();  // dlogits may be the logits: every lane has read what it needs before the first one writes
        float x[NV], mx = kNegInf;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = FULL || lane + 32 * i < E ? to_f32(raw[i]) : kNegInf;
            mx = fmaxf(mx, x[i]);
        }
        mx = warp_max(mx);
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = exp2_approx((x[i] - mx) * kLog2e);
            sum += x[i];
            dot = fmaf(x[i], base[i], dot);
        }
        const float inv = rcp_approx(warp_sum(sum));
        const float pj = mine ? exp2_approx((my_logit - mx) * kLog2e) * inv : 0.0f;
        float g = mine ? gw : 0.0f;
        if (p.renorm && p.dweights) {
            // weights = p / S over the choices: d/dp = (gw - sum gw * weights) / S
            const float s = warp_sum(pj), gp = warp_sum(g * pj);
            const float inv_s = rcp_approx(s);
            g = (g - gp * inv_s) * inv_s;
        }
        dot = warp_sum(fmaf(dot, inv, mine ? pj * g : 0.0f));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (FULL || lane + 32 * i < E) out[lane + 32 * i] = from_f32<T>(x[i] * inv * (base[i] - dot));
        __syncwarp();
        if (mine) out[my] = from_f32<T>(pj * (s_base[my] + g - dot));
    }
}

bool is_float_type(int dtype) { return dtype == ASCB200_F32 || dtype == ASCB200_F16 || dtype == ASCB200_BF16; }
bool element_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int route_blocks(int tokens) { return static_cast<int>(std::min<long long>((tokens + kRouteWarps - 1ll) / kRouteWarps, kMaxRouteBlocks)); }
size_t route_workspace(int tokens, int experts)
{
    if (tokens <= 0 || experts <= 0) return 0;
    const int blocks = route_blocks(tokens);
    return blocks == 1 ? 0 : static_cast<size_t>(blocks) * (2 * static_cast<size_t>(experts) + 1) * 4;
}

template <typename T, int NV, bool FULL>
int launch_route_as(const RouteArgs& p, int blocks, cudaStream_t st)
{
    const size_t smem = (kRouteWarps + 1) * static_cast<size_t>(p.experts) * 4;
    if (smem > 46 * 1024) {  // more than 692 experts: beyond what a launch may take unasked
        static bool configured[16] = {};
        int dev = 0;
        ASCB200_CUDA(cudaGetDevice(&dev));
        if (!configured[dev & 15]) {
            ASCB200_CUDA(cudaFuncSetAttribute(route_kernel<T, NV, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (kRouteWarps + 1) * kMaxExperts * 4));
            configured[dev & 15] = true;
        }
    }
    ASCB200_CUDA(launch_pdl(route_kernel<T, NV, FULL>, blocks, kRouteWarps * 32, smem, st, p));
    if (blocks > 1) ASCB200_CUDA(launch_pdl(route_finish_kernel, kFinishBlocks, kFinishWarps * 32, 0, st, p, blocks));
    return ASCB200_OK;
}
template <typename T, int NV>
int launch_route_nv(const RouteArgs& p, int blocks, cudaStream_t st)
{
    return p.experts == 32 * NV ? launch_route_as<T, NV, true>(p, blocks, st) : launch_route_as<T, NV, false>(p, blocks, st);
}
template <typename T>
int launch_route(const RouteArgs& p, int blocks, cudaStream_t st)
{
    if (p.experts <= 32) return launch_route_nv<T, 1>(p, blocks, st);
    if (p.experts <= 64) return launch_route_nv<T, 2>(p, blocks, st);
    if (p.experts <= 128) return launch_route_nv<T, 4>(p, blocks, st);
    if (p.experts <= 256) return launch_route_nv<T, 8>(p, blocks, st);
    if (p.experts <= 512) return launch_route_nv<T, 16>(p, blocks, st);
    return launch_route_nv<T, 32>(p, blocks, st);
}

template <typename T, int NV>
int launch_route_grad_as(const RouteGradArgs& p, int sms, cudaStream_t st)
{
    const int blocks = static_cast<int>(std::min((p.tokens + 7ll) / 8, 8ll * sms));
    const size_t smem = static_cast<size_t>(p.experts) * 4;
    if (p.experts == 32 * NV) ASCB200_CUDA(launch_pdl(route_grad_kernel<T, NV, true>, blocks, 256, smem, st, p));
    else ASCB200_CUDA(launch_pdl(route_grad_kernel<T, NV, false>, blocks, 256, smem, st, p));
    return ASCB200_OK;
}
template <typename T>
int launch_route_grad(const RouteGradArgs& p, int sms, cudaStream_t st)
{
    if (p.experts <= 32) return launch_route_grad_as<T, 1>(p, sms, st);
    if (p.experts <= 64) return launch_route_grad_as<T, 2>(p, sms, st);
    if (p.experts <= 128) return launch_route_grad_as<T, 4>(p, sms, st);
    if (p.experts <= 256) return launch_route_grad_as<T, 8>(p, sms, st);
    if (p.experts <= 512) return launch_route_grad_as<T, 16>(p, sms, st);
    return launch_route_grad_as<T, 32>(p, sms, st);
}

// Sizes and types that ascb200_route and ascb200_route_grad share.
int check_route(int tokens, int experts, int top_k, int dtype, int64_t& ld, int renorm)
{
    if (tokens < 0 || experts <= 0 || top_k <= 0 || top_k > experts || (renorm != 0 && renorm != 1)) return ASCB200_EINVAL;
    if (experts > kMaxExperts || top_k > kMaxTopK) return ASCB200_ETOOBIG;
    if (!is_float_type(dtype)) return ASCB200_EUNSUPPORTED;
    if (ld == 0) ld = experts;
    return ld < experts ? ASCB200_EINVAL : ASCB200_OK;
}

int run_route(const ascb200_route_desc* desc, cudaStream_t stream)
{
    DeviceState* st = current_state();
    if (!st) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_route_desc d = *desc;
    const int rc = check_route(d.tokens, d.experts, d.top_k, d.dtype, d.ld_logits, d.renorm);
    if (rc != ASCB200_OK) return rc;
    if (d.reserved != 0) return ASCB200_EINVAL;
    if (!element_aligned(d.counts_dev, 8) || !element_aligned(d.num_tokens_dev, 8) || !element_aligned(d.prob_mean_dev, 4) || !element_aligned(d.loss_dev, 4))
        return ASCB200_EALIGN;
    if (d.tokens == 0) {  // nothing was routed
        if (d.counts_dev) ASCB200_CUDA(cudaMemsetAsync(d.counts_dev, 0, static_cast<size_t>(d.experts) * 8, stream));
        if (d.num_tokens_dev) ASCB200_CUDA(cudaMemsetAsync(d.num_tokens_dev, 0, 8, stream));
        if (d.prob_mean_dev) ASCB200_CUDA(cudaMemsetAsync(d.prob_mean_dev, 0, static_cast<size_t>(d.experts) * 4, stream));
        if (d.loss_dev) ASCB200_CUDA(cudaMemsetAsync(d.loss_dev, 0, 4, stream));
        return ASCB200_OK;
    }
    if (!d.logits_dev || !d.idx_dev || !d.weights_dev) return ASCB200_EINVAL;
    if (!element_aligned(d.logits_dev, d.dtype == ASCB200_F32 ? 4 : 2) || !element_aligned(d.idx_dev, 4) || !element_aligned(d.weights_dev, 4)) return ASCB200_EALIGN;
    const size_t need = route_workspace(d.tokens, d.experts);
    if (need > 0 && (!d.workspace_dev || d.workspace_bytes < need)) return ASCB200_EINVAL;
    if (need > 0 && !aligned_to(d.workspace_dev, 16)) return ASCB200_EALIGN;
    RouteArgs p = {};
    p.logits = d.logits_dev, p.valid = d.valid_dev, p.idx = d.idx_dev, p.weights = d.weights_dev;
    p.counts = reinterpret_cast<long long*>(d.counts_dev), p.num_tokens = reinterpret_cast<long long*>(d.num_tokens_dev);
    p.prob_mean = d.prob_mean_dev, p.loss = d.loss_dev;
    p.ld = d.ld_logits, p.tokens = d.tokens, p.experts = d.experts, p.top_k = d.top_k, p.renorm = d.renorm;
    const int blocks = std::min(route_blocks(d.tokens), std::max(2, 2 * st->sm_count));
    if (need > 0) {
        p.part_prob = static_cast<float*>(d.workspace_dev);
        p.part_count = reinterpret_cast<int*>(p.part_prob + static_cast<size_t>(blocks) * d.experts);
        p.part_tokens = p.part_count + static_cast<size_t>(blocks) * d.experts;
    }
    switch (d.dtype) {
        case ASCB200_F16: return launch_route<__half>(p, blocks, stream);
        case ASCB200_BF16: return launch_route<__nv_bfloat16>(p, blocks, stream);
        default: return launch_route<float>(p, blocks, stream);
    }
}

int run_route_grad(const ascb200_route_grad_desc* desc, cudaStream_t stream)
{
    DeviceState* st = current_state();
    if (!st) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_route_grad_desc d = *desc;
    int rc = check_route(d.tokens, d.experts, d.top_k, d.dtype, d.ld_logits, d.renorm);
    if (rc != ASCB200_OK) return rc;
    if (d.ld_dlogits == 0) d.ld_dlogits = d.experts;
    if (d.ld_dlogits < d.experts || d.reserved != 0) return ASCB200_EINVAL;
    if (d.tokens == 0) return ASCB200_OK;
    if (!d.logits_dev || !d.idx_dev || !d.dlogits_dev || (d.dlogits_dev == d.logits_dev && d.ld_dlogits != d.ld_logits)) return ASCB200_EINVAL;
    if (d.dloss_dev && (!d.counts_dev || !d.num_tokens_dev)) return ASCB200_EINVAL;
    const int esz = d.dtype == ASCB200_F32 ? 4 : 2;
    if (!element_aligned(d.logits_dev, esz) || !element_aligned(d.dlogits_dev, esz) || !element_aligned(d.idx_dev, 4) || !element_aligned(d.counts_dev, 8) ||
        !element_aligned(d.num_tokens_dev, 8) || !element_aligned(d.dloss_dev, 4) || !element_aligned(d.dweights_dev, 4))
        return ASCB200_EALIGN;
    RouteGradArgs p = {};
    p.logits = d.logits_dev, p.idx = d.idx_dev, p.counts = reinterpret_cast<const long long*>(d.counts_dev);
    p.num_tokens = reinterpret_cast<const long long*>(d.num_tokens_dev), p.dloss = d.dloss_dev, p.dweights = d.dweights_dev, p.dlogits = d.dlogits_dev;
    p.ld = d.ld_logits, p.ld_out = d.ld_dlogits, p.tokens = d.tokens, p.experts = d.experts, p.top_k = d.top_k, p.renorm = d.renorm;
    const int sms = st->sm_count;
    switch (d.dtype) {
        case ASCB200_F16: return launch_route_grad<__half>(p, sms, stream);
        case ASCB200_BF16: return launch_route_grad<__nv_bfloat16>(p, sms, stream);
        default: return launch_route_grad<float>(p, sms, stream);
    }
}

}  // namespace
}  // namespace ascb200

extern "C" {

size_t ascb200_route_workspace_bytes(int32_t tokens, int32_t experts) { return ascb200::route_workspace(tokens, experts); }

int ascb200_route(const ascb200_route_desc* desc, void* stream) { return ascb200::run_route(desc, static_cast<cudaStream_t>(stream)); }

int ascb200_route_grad(const ascb200_route_grad_desc* desc, void* stream) { return ascb200::run_route_grad(desc, static_cast<cudaStream_t>(stream)); }

}  // extern "C"
