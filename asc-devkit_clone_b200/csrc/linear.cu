// Linear layers: matrix product with bias, activation and residual in its output stage, and its gradients.
//
//   y = act(z) + residual,   z = x w^T (int8: scaled per token and channel) + bias
//
// Many rows run on the tensor-core GEMM kernels with the output stage of a linear layer (gemm_linear.cu).  A few tokens run here:
// the product then reads every weight once and is memory bound.
//
// Gradients: dz = dy * act'(z) and dbias = sum over rows of dz in one pass over dy and z, then dx = dz w and dw = dz^T x as plain GEMMs; of a few
// rows all in one launch.
#include <algorithm>
#include <type_traits>

#include "activation.cuh"
#include "gemm_host.cuh"
#include "partial_sum.cuh"

namespace ascb200 {
namespace {

// ---- a few tokens ----------------------------------------------------------------------------------------------------------
// The weights' rows are the 16-row operand of mma.sync m16n8 and the tokens its eight columns, so that every weight that comes from
// memory is used by one instruction for all tokens.  A sum over k does not care for the order of k as long as both operands agree,
// so a lane feeds the instructions straight from 16 contiguous bytes of a weight row (its first two words are the lane's k slots of
// one instruction, the last two those of the next): 64 bytes of a row per pair of instructions, no shuffles and no shared memory.
//
// Two or three blocks per SM, all resident, each with an equal run of weight rows, one to three tiles of 16 in a pass: what is loaded of
// the tokens serves every tile of the pass.  A block's eight warps take 256-byte pieces of the rows in turn and add their sums in warp
// order through shared memory at the end of the pass.
constexpr int kRowsTokens = 16;       // per block
constexpr int kRowsTile = 16;
constexpr int kRowsWarps = 8;
constexpr int kRowsUnroll = 4;        // 64-byte chunks per warp and step
constexpr int kRowsBlocksPerSm(int groups) { return groups == 1 ? 3 : 2; }  // by groups of eight tokens: what registers allow

struct RowsArgs {
    const uint8_t* x;
    const uint8_t* w;
    const float* tok;
    const float* ch;
    const void* bias;
    const void* residual;
    void* y;
    void* z;
    long long ldx, ldw;  // bytes
    long long ld_residual, ldy, ldz;
    int m, n, k_bytes;
    int bias_f32, act;
};

template <int KIND>
__device__ __forceinline__ void mma_16x8(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (KIND == ASCB200_KIND_S8) {
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        float* f = reinterpret_cast<float*>(c);
        if constexpr (KIND == ASCB200_KIND_F16)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                         : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                         : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                         : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

template <int KIND>
__device__ __forceinline__ uint32_t add_bits(uint32_t a, uint32_t b)
{
    return KIND == ASCB200_KIND_S8 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

// 16 bytes at `off` of a row of `bytes` bytes; what lies behind its end reads as zero and is not touched.  STREAM: read once.
template <bool STREAM>
__device__ __forceinline__ uint4 load_piece(const uint8_t* row, int off, int bytes)
{
    uint4 r = make_uint4(0u, 0u, 0u, 0u);
    if (off + 16 <= bytes) {
        if constexpr (STREAM)
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(row + off));
        else
            r = __ldg(reinterpret_cast<const uint4*>(row + off));
    } else if (off < bytes) {
        uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 15; ++j)
            if (off + j < bytes) u[j >> 2] |= static_cast<uint32_t>(__ldg(row + off + j)) << (8 * (j & 3));
        r = make_uint4(u[0], u[1], u[2], u[3]);
    }
    return r;
}

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <int KIND, int NT, int R, typename OT>  // NT: groups of eight tokens; R: tiles of 16 rows per pass
__global__ void __launch_bounds__(kRowsWarps * 32, kRowsBlocksPerSm(NT))
linear_rows_kernel(const RowsArgs p)
{
    constexpr int STEP = kRowsUnroll * 64;
    constexpr int CHAINS = NT == 1 ? 2 : 1;  // independent chains of instructions per tile: two in either case
    __shared__ uint32_t part[kRowsWarps][NT * 8][R * kRowsTile + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, q = lane & 3;
    const int token0 = blockIdx.y * kRowsTokens, tokens = min(kRowsTokens, p.m - token0);
    const uint8_t* xs = p.x + token0 * p.ldx;
    const int row0 = static_cast<int>(static_cast<long long>(blockIdx.x) * p.n / gridDim.x);
    const int row1 = static_cast<int>((static_cast<long long>(blockIdx.x) + 1) * p.n / gridDim.x);
    // While the kernel before this one drains, ask L2 for the warp's first pieces (hints: nothing is read into the program yet).
    if (row0 + lane < row1 && warp * STEP < p.k_bytes) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p.w + (row0 + lane) * p.ldw + warp * STEP));
        if (warp * STEP + 128 < p.k_bytes) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.w + (row0 + lane) * p.ldw + warp * STEP + 128));
    }
    grid_dependency_wait();
    for (int n0 = row0; n0 < row1; n0 += R * kRowsTile) {
        const int tiles = min(R, (row1 - n0 + kRowsTile - 1) / kRowsTile);
        uint32_t acc[R][NT][CHAINS][4] = {};
        for (int base = warp * STEP; base < p.k_bytes; base += kRowsWarps * STEP) {
            uint4 x[NT][kRowsUnroll];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r >= tiles) break;  // the same for the whole block
                const int n = n0 + r * kRowsTile + g;
                const uint8_t* w0 = p.w + n * p.ldw;
                const uint8_t* w1 = w0 + 8 * p.ldw;
                const int bytes0 = n < row1 ? p.k_bytes : 0, bytes1 = n + 8 < row1 ? p.k_bytes : 0;  // rows behind the run count as empty
                uint4 a[kRowsUnroll], b[kRowsUnroll];
#pragma unroll
                for (int u = 0; u < kRowsUnroll; ++u) {
                    const int off = base + u * 64 + q * 16;
                    a[u] = load_piece<true>(w0, off, bytes0);
                    b[u] = load_piece<true>(w1, off, bytes1);
                }
                if (r == 0) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int u = 0; u < kRowsUnroll; ++u) {
                            x[t][u] = make_uint4(0u, 0u, 0u, 0u);
                            if (t * 8 + g < tokens) x[t][u] = load_piece<false>(xs + (t * 8 + g) * p.ldx, base + u * 64 + q * 16, p.k_bytes);
                        }
                }
#pragma unroll
                for (int u = 0; u < kRowsUnroll; ++u)
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        mma_16x8<KIND>(acc[r][t][0], a[u].x, b[u].x, a[u].y, b[u].y, x[t][u].x, x[t][u].y);
                        mma_16x8<KIND>(acc[r][t][CHAINS - 1], a[u].z, b[u].z, a[u].w, b[u].w, x[t][u].z, x[t][u].w);
                    }
            }
        }
        // accumulators: rows g and g + 8, tokens 2 q and 2 q + 1
        if (n0 > row0) __syncthreads();  // the pass before has been read
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[warp][t * 8 + 2 * q + (j & 1)][r * kRowsTile + g + (j >> 1) * 8] = CHAINS == 2 ? add_bits<KIND>(acc[r][t][0][j], acc[r][t][CHAINS - 1][j]) : acc[r][t][0][j];
        __syncthreads();
        constexpr int cols = R * kRowsTile;
        for (int i = threadIdx.x; i < NT * 8 * cols; i += kRowsWarps * 32) {
            const int local = i / cols, token = token0 + local, col = i % cols, n = n0 + col;
            if (local >= tokens || n >= row1) continue;
            float f;
            if constexpr (KIND == ASCB200_KIND_S8) {
                int s = 0;
#pragma unroll
                for (int v = 0; v < kRowsWarps; ++v) s += static_cast<int>(part[v][local][col]);
                f = static_cast<float>(s) * p.ch[n];
                if (p.tok) f *= p.tok[token];
            } else {
                f = 0.0f;
#pragma unroll
                for (int v = 0; v < kRowsWarps; ++v) f += __uint_as_float(part[v][local][col]);
            }
            if (p.bias) f += p.bias_f32 ? static_cast<const float*>(p.bias)[n] : as_f32(static_cast<const OT*>(p.bias)[n]);
            if (p.z) static_cast<OT*>(p.z)[token * p.ldz + n] = rounded<OT>(f);
            ASCB200_ACT_SWITCH(p.act, { f = act::value<ACT>(f); })
            if (p.residual) f += as_f32(static_cast<const OT*>(p.residual)[token * p.ld_residual + n]);
            static_cast<OT*>(p.y)[token * p.ldy + n] = rounded<OT>(f);
        }
    }
}

template <int KIND, int NT, int R, typename OT>
int launch_rows_as(const RowsArgs& p, dim3 grid, cudaStream_t st)
{
    ASCB200_CUDA(launch_pdl(linear_rows_kernel<KIND, NT, R, OT>, grid, kRowsWarps * 32, 0, st, p));
    return ASCB200_OK;
}
// How a call is cut for the kernel above: blocks of 16 tokens (grid.y) times runs of weight rows.  A run has at least as many rows as a block
// has tokens: with fewer, the tokens would be read more often than the weights.
struct RowsCut {
    int groups, by_tokens, runs, tiles, steps;  // tiles of 16 rows per run; 2048-byte steps of a block along k
};
RowsCut cut_rows(int m, int n, int64_t k_bytes, int sms)
{
    RowsCut c;
    c.groups = m <= 8 ? 1 : 2;
    c.by_tokens = (m + kRowsTokens - 1) / kRowsTokens;
    c.runs = std::max(1, std::min(n / (8 * c.groups), kRowsBlocksPerSm(c.groups) * sms / c.by_tokens));
    c.tiles = ((n + c.runs - 1) / c.runs + kRowsTile - 1) / kRowsTile;
    c.steps = static_cast<int>((k_bytes + kRowsWarps * kRowsUnroll * 64 - 1) / (kRowsWarps * kRowsUnroll * 64));
    return c;
}
// Up to 16 tokens the kernel above is the faster one at every size measured (us, bf16, m x n x k, weights in L2: 1 x 4096 x 4096 6.7, 16 x 4096 x 4096 8.5 against
// 12.8 on the GEMM kernels at 17 rows, 16 x 11008 x 4096 19.5 against 21.4, 16 x 512 x 512 2.4 against 5.8; weights from memory: 8.4, 10.8 against 13.7,
// 21.1 against 24.2 at 32 rows).  Up to 256, while every block has one
// or two tiles and a short k, it still is: 128 x 512 x 512 2.7 against 5.9, 256 x 256 x 4096 8.0 against 10.3, 32 x 4096 x 1024 5.6 against
// 9.4, 64 x 2048 x 2048 8.1 against 9.0; but 32 x 4096 x 4096 (two tiles, four steps) 13.8 against 12.5, 64 x 4096 x 256 (four tiles) 8.7 against 5.7.
bool rows_suit(int m, int n, int64_t k_bytes, int sms)
{
    if (k_bytes > (1ll << 30)) return false;  // offsets within a row are 32-bit
    if (m <= kRowsTokens) return true;
    if (m > 256) return false;
    const RowsCut c = cut_rows(m, n, k_bytes, sms);
    return c.tiles <= 2 && c.tiles * c.tiles * c.steps <= 8;
}

template <int KIND, typename OT>
int launch_rows_of(const RowsArgs& p, int sms, cudaStream_t st)
{
    const RowsCut c = cut_rows(p.m, p.n, p.k_bytes, sms);
    const dim3 grid(c.runs, c.by_tokens);
    // One tile per pass for runs that have no more: the registers of the others would spill (16 x 4096 x 4096 bf16 8.9 against 10.3 us, 1 x 4096 x
    // 11008 17.0 against 18.1); longer runs share the tokens' loads between tiles (16 x 11008 x 4096: 30.9 us with one, 20.2 with three).
    if (c.groups == 1) return c.tiles == 1 ? launch_rows_as<KIND, 1, 1, OT>(p, grid, st) : launch_rows_as<KIND, 1, 2, OT>(p, grid, st);
    return c.tiles == 1 ? launch_rows_as<KIND, 2, 1, OT>(p, grid, st) : launch_rows_as<KIND, 2, 3, OT>(p, grid, st);
}
template <int KIND>
int launch_rows(const RowsArgs& p, int y_dtype, int sms, cudaStream_t st)
{
    if (y_dtype == ASCB200_F16) return launch_rows_of<KIND, __half>(p, sms, st);
    if (y_dtype == ASCB200_BF16) return launch_rows_of<KIND, __nv_bfloat16>(p, sms, st);
    return launch_rows_of<KIND, float>(p, sms, st);
}

bool element_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool operand_aligned(const void* p, int64_t ld, int bytes) { return aligned_to(p, 16) && (ld * bytes) % 16 == 0; }
int float_bytes(int dtype) { return dtype == ASCB200_F32 ? 4 : 2; }
bool is_float_type(int dtype) { return dtype == ASCB200_F32 || dtype == ASCB200_F16 || dtype == ASCB200_BF16; }

int run_linear(const ascb200_linear_desc* desc, cudaStream_t stream)
{
    DeviceState* state = current_state();
    if (!state) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_linear_desc d = *desc;
    if (d.m < 0 || d.n < 0 || d.k <= 0 || d.reserved != 0 || (d.trans_w != 0 && d.trans_w != 1)) return ASCB200_EINVAL;
    if (d.act < ASCB200_ACT_NONE || d.act > ASCB200_ACT_SILU) return ASCB200_EINVAL;
    if (d.kind != ASCB200_KIND_F16 && d.kind != ASCB200_KIND_BF16 && d.kind != ASCB200_KIND_S8) return ASCB200_EUNSUPPORTED;
    const bool s8 = d.kind == ASCB200_KIND_S8;
    const int own = d.kind == ASCB200_KIND_F16 ? ASCB200_F16 : ASCB200_BF16;
    if (s8 ? !is_float_type(d.y_dtype) : d.y_dtype != own && d.y_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    if (s8 && d.z_dev) return ASCB200_EUNSUPPORTED;
    if (!s8 && (d.tok_scale_dev || d.ch_scale_dev)) return ASCB200_EINVAL;
    if (d.bias_dev && d.bias_dtype != ASCB200_F32 && d.bias_dtype != d.y_dtype) return ASCB200_EUNSUPPORTED;
    if (d.ldx == 0) d.ldx = d.k;
    if (d.ldw == 0) d.ldw = d.trans_w ? d.k : d.n;
    if (d.ld_residual == 0) d.ld_residual = d.n;
    if (d.ldy == 0) d.ldy = d.n;
    if (d.ldz == 0) d.ldz = d.n;
    if (d.ldx < d.k || d.ldw < (d.trans_w ? d.k : d.n) || d.ld_residual < d.n || d.ldy < d.n || d.ldz < d.n) return ASCB200_EINVAL;
    if (d.m == 0 || d.n == 0) return ASCB200_OK;
    if (!d.x_dev || !d.w_dev || !d.y_dev || (s8 && !d.ch_scale_dev) || d.y_dev == d.z_dev) return ASCB200_EINVAL;
    if (d.residual_dev && ((d.y_dev == d.residual_dev && d.ldy != d.ld_residual) || d.z_dev == d.residual_dev)) return ASCB200_EINVAL;
    const int esz = s8 ? 1 : 2, osz = float_bytes(d.y_dtype);
    if (!operand_aligned(d.x_dev, d.ldx, esz) || !operand_aligned(d.w_dev, d.ldw, esz)) return ASCB200_EALIGN;
    if (!element_aligned(d.y_dev, osz) || !element_aligned(d.z_dev, osz) || !element_aligned(d.residual_dev, osz) || !element_aligned(d.tok_scale_dev, 4) ||
        !element_aligned(d.ch_scale_dev, 4) || (d.bias_dev && !element_aligned(d.bias_dev, float_bytes(d.bias_dtype))))
        return ASCB200_EALIGN;

    if (d.trans_w && rows_suit(d.m, d.n, static_cast<int64_t>(d.k) * esz, state->sm_count)) {
        RowsArgs p = {};
        p.x = static_cast<const uint8_t*>(d.x_dev), p.w = static_cast<const uint8_t*>(d.w_dev), p.tok = d.tok_scale_dev, p.ch = d.ch_scale_dev;
        p.bias = d.bias_dev, p.residual = d.residual_dev, p.y = d.y_dev, p.z = d.z_dev;
        p.ldx = d.ldx * esz, p.ldw = d.ldw * esz, p.ld_residual = d.ld_residual, p.ldy = d.ldy, p.ldz = d.ldz;
        p.m = d.m, p.n = d.n, p.k_bytes = d.k * esz, p.bias_f32 = d.bias_dtype == ASCB200_F32, p.act = d.act;
        if (s8) return launch_rows<ASCB200_KIND_S8>(p, d.y_dtype, state->sm_count, stream);
        if (d.kind == ASCB200_KIND_F16) return launch_rows<ASCB200_KIND_F16>(p, d.y_dtype, state->sm_count, stream);
        return launch_rows<ASCB200_KIND_BF16>(p, d.y_dtype, state->sm_count, stream);
    }

    ascb200_gemm_desc q = {};
    q.kind = d.kind, q.m = d.m, q.n = d.n, q.k = d.k;
    q.a_dev = d.x_dev, q.lda = d.ldx, q.b_dev = d.w_dev, q.ldb = d.ldw, q.trans_b = d.trans_w;
    q.c_dev = d.y_dev, q.ldc = d.ldy, q.c_dtype = d.y_dtype;
    q.c2_dev = d.z_dev, q.ldc2 = d.ldz, q.c2_dtype = d.y_dtype;
    q.epilogue = s8 ? ASCB200_EPI_DEQUANT_TOKEN_CHANNEL : ASCB200_EPI_CAST;
    q.tok_scale_dev = d.tok_scale_dev, q.ch_scale_dev = d.ch_scale_dev;
    const gemm::LinearArgs lin = {d.bias_dev, d.bias_dtype == ASCB200_F32, d.act, d.residual_dev, d.ld_residual};
    return gemm::run_gemm(&q, nullptr, 0, stream, nullptr, &lin);
}

// ---- gradients --------------------------------------------------------------------------------------------------------------
// dz = dy * act'(z), rounded to the operands' type for the two products that follow (the rounding that any 16-bit product of it
// needs: beside the rounding of the results it raises their error from 0.0017 to 0.0023 of their size in bf16, 0.00021 to 0.00029 in fp16; with dz as two
// numbers both products would have twice the work); dbias from the fp32 values before that rounding.  A thread owns eight columns and walks down rows; memory bound.
struct ActGradArgs {
    const void* dy;
    const void* z;
    void* dz;
    float* partial;  // [row blocks][n], or nullptr
    void* dbias;     // a single block of rows writes it itself
    long long ld_dy, ldz, ld_dz;
    int m, n, dbias_f32;
};

template <typename T>
struct alignas(16) Eight {
    T e[8];
};
// VEC (rows of dy, z and dz start on 16 bytes and n is a multiple of 8): a lane's eight columns are neighbours.  Else they are 32 apart, so
// that a warp's accesses of one element each are contiguous.  (One kernel that chose per row took 64 us for 4096 x 11008, and 117 with
// four rows in flight: the two paths' loads met in the same registers and were waited for one by one.)
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int col, int n, Eight<T>& r)
{
    if constexpr (VEC) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + col));
        r = *reinterpret_cast<const Eight<T>*>(&v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r.e[j] = col + 32 * j < n ? row[col + 32 * j] : rounded<T>(0.0f);
    }
}

template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256)
act_grad_kernel(const ActGradArgs p)
{
    __shared__ float part[8][256];
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int in_block = VEC ? lane * 8 : lane, col = blockIdx.x * 256 + in_block;
    float acc[8] = {};
    constexpr int U = 4;  // rows whose loads are in flight together
    if (col < p.n) {
        const long long step = static_cast<long long>(gridDim.y) * 8;
        for (long long row0 = static_cast<long long>(blockIdx.y) * 8 + warp; row0 < p.m; row0 += U * step) {
            Eight<T> dyr[U], zr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = min(row0 + u * step, static_cast<long long>(p.m) - 1);
                load8<T, VEC>(static_cast<const T*>(p.dy) + row * p.ld_dy, col, p.n, dyr[u]);
                if constexpr (ACT != ASCB200_ACT_NONE) load8<T, VEC>(static_cast<const T*>(p.z) + row * p.ldz, col, p.n, zr[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long row = row0 + u * step;
                if (row >= p.m) break;
                float dy[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) dy[j] = as_f32(dyr[u].e[j]);
                if constexpr (ACT != ASCB200_ACT_NONE) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) dy[j] *= act::slope<ACT>(as_f32(zr[u].e[j]));
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] += dy[j];
                if (p.dz) {
                    T* out = static_cast<T*>(p.dz) + row * p.ld_dz + col;
                    if constexpr (VEC) {
                        Eight<T> v;
#pragma unroll
                        for (int j = 0; j < 8; ++j) v.e[j] = rounded<T>(dy[j]);
                        *reinterpret_cast<Eight<T>*>(out) = v;
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (col + 32 * j < p.n) out[32 * j] = rounded<T>(dy[j]);
                    }
                }
            }
        }
    }
    if (!p.partial) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) part[warp][in_block + (VEC ? j : 32 * j)] = acc[j];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < p.n) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += part[i][threadIdx.x];
        if (gridDim.y > 1) p.partial[static_cast<size_t>(blockIdx.y) * p.n + c] = v;
        else if (p.dbias_f32) static_cast<float*>(p.dbias)[c] = v;
        else static_cast<T*>(p.dbias)[c] = rounded<T>(v);
    }
}

template <typename T, bool VEC>
int launch_act_grad_as(const ActGradArgs& p, int act, dim3 grid, cudaStream_t st)
{
    switch (act) {
#define ASCB200_ACT_GRAD(A) case A: ASCB200_CUDA(launch_pdl(act_grad_kernel<T, A, VEC>, grid, 256, 0, st, p)); return ASCB200_OK;
        ASCB200_ACT_GRAD(ASCB200_ACT_FASTER_GELU)
        ASCB200_ACT_GRAD(ASCB200_ACT_RELU)
        ASCB200_ACT_GRAD(ASCB200_ACT_GELU)
        ASCB200_ACT_GRAD(ASCB200_ACT_GELU_TANH)
        ASCB200_ACT_GRAD(ASCB200_ACT_SILU)
        default: ASCB200_CUDA(launch_pdl(act_grad_kernel<T, ASCB200_ACT_NONE, VEC>, grid, 256, 0, st, p)); return ASCB200_OK;
#undef ASCB200_ACT_GRAD
    }
}

template <typename T>
int launch_act_grad(const ActGradArgs& p, int act, bool vec, dim3 grid, cudaStream_t st)
{
    return vec ? launch_act_grad_as<T, true>(p, act, grid, st) : launch_act_grad_as<T, false>(p, act, grid, st);
}

// ---- gradients of a few rows ----------------------------------------------------------------------------------------------------
// Up to 16 rows everything fits one launch, whose blocks have one of three jobs.  What bounds it is reading w once and writing dw once.
//   dx    a strip of 64 columns of w; its rows are shared by the blocks of a cluster, and within a block by the warps, 16 at a time.  The sums
//         meet in shared memory, of the block and then of the cluster, always in the same order.
//   dw    tiles of 64 x 256: one instruction per 16 x 8 outputs sums all rows.
//   dbias 256 columns.
// Each job makes the dz that it needs itself, as the sum of two numbers of the operands' type: with so few terms in a sum, a single rounding of dz would
// show beside that of the result (1 x 64 x 64: the error of dw up to twice as large), and the matrix instructions have the time.
//
// As in the kernel for a few tokens, the order of the summands and of the columns is free as long as the operands agree.  dx: lane (g, q) reads
// 16 bytes, columns 8 g .. 8 g + 7, of rows 4 q .. 4 q + 3; the i-th of eight instructions takes the i-th of each lane's columns, two
// rows packed by one byte permutation.  dw: the columns of an instruction are those that leave a lane with eight neighbours after four.
//
// One launch instead of four, of which two are GEMMs of mostly empty tiles (us, bf16 silu with dbias, n x k, 16 rows here against 17 on the GEMMs: 320 x 481
// 5.8 / 11.1, 1792 x 3864 16.9 / 25.6, 4096 x 4096 26.8 / 30.4, 11008 x 4096 58.8 / 60.3, 4096 x 11008 56.5 / 60; one row of 11008 x 4096 52.7, 3.4 TB/s;
// the second part of dz takes 5 to 10 % of that, keeping infinities from it 3 %).  What keeps it from the memory's rate is the latency of a block's loads: dx alone of
// 1 x 11008 x 4096 runs at 3.6 TB/s, dw alone at 4.6; 128 registers per thread leave room for two blocks per SM.
constexpr int kGradRows = 16;
constexpr int kGradThreads = 256, kGradWarps = 8;
constexpr int kGradStrip = 64;                         // columns of dx per cluster
constexpr int kGradTileRows = 64, kGradTileCols = 256;  // of dw
constexpr int kPartLd = kGradStrip + 8;

struct GradRowsArgs {
    const void* dy;
    const void* z;
    const void* x;
    const void* w;
    void* dx;
    void* dw;
    void* dbias;
    long long ld_dy, ldz, ldx, ldw, ld_dx, ld_dw;
    int m, n, k;
    int dw_f32, dbias_f32;
    int quads;   // four elements of dy and z from a column that is a multiple of four start on 8 bytes
    int dw_vec;  // eight elements of dw from a column that is a multiple of eight start on 16 bytes, and k is a multiple of eight
    int splits;  // blocks per cluster
    int dx_blocks, dw_blocks;
};

// Four neighbouring 16-bit elements from column c on, zeros from column n on.
__device__ __forceinline__ uint2 load_quad(const uint16_t* row, int c, int n, bool aligned)
{
    if (aligned && c + 4 <= n) return __ldg(reinterpret_cast<const uint2*>(row + c));
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < n ? __ldg(row + c + j) : 0u;
    return make_uint2(v[0] | (v[1] << 16), v[2] | (v[3] << 16));
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v)
{
    T e[2];
    *reinterpret_cast<uint32_t*>(e) = v;
    return make_float2(as_f32(e[0]), as_f32(e[1]));
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b)
{
    T e[2] = {rounded<T>(a), rounded<T>(b)};
    return *reinterpret_cast<uint32_t*>(e);
}
struct RawQuad {
    uint2 dy, z;
};
template <int ACT>
__device__ __forceinline__ RawQuad load_dz(const GradRowsArgs& p, int t, int c)
{
    RawQuad r = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    if (t < p.m) {
        r.dy = load_quad(static_cast<const uint16_t*>(p.dy) + t * p.ld_dy, c, p.n, p.quads);
        if constexpr (ACT != ASCB200_ACT_NONE) r.z = load_quad(static_cast<const uint16_t*>(p.z) + t * p.ldz, c, p.n, p.quads);
    }
    return r;
}
// dz = high + low; the slopes of no activation and of RELU leave dy as it is, or nothing.
template <int ACT>
constexpr bool exact_dz() { return ACT == ASCB200_ACT_NONE || ACT == ASCB200_ACT_RELU; }
template <typename T>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& high, uint32_t& low)
{
    high = pack_pair<T>(a, b);
    const float2 h = unpack_pair<T>(high);
    // (an infinity or NaN is in `high`; fp16 saturates, and what is beyond stays out of `low` as it does of dz)
    const float la = a - h.x, lb = b - h.y;
    low = pack_pair<T>(fabsf(la) <= fabsf(h.x) * 0.00390625f ? la : 0.0f, fabsf(lb) <= fabsf(h.y) * 0.00390625f ? lb : 0.0f);
}
template <typename T, int ACT>
__device__ __forceinline__ uint2 dz_of(const RawQuad& r, uint2& low)
{
    low = make_uint2(0u, 0u);
    if constexpr (ACT == ASCB200_ACT_NONE) return r.dy;
    const float2 a = unpack_pair<T>(r.dy.x), b = unpack_pair<T>(r.dy.y), za = unpack_pair<T>(r.z.x), zb = unpack_pair<T>(r.z.y);
    uint2 high;
    if constexpr (exact_dz<ACT>()) {
        high = make_uint2(pack_pair<T>(a.x * act::slope<ACT>(za.x), a.y * act::slope<ACT>(za.y)), pack_pair<T>(b.x * act::slope<ACT>(zb.x), b.y * act::slope<ACT>(zb.y)));
    } else {
        split_pair<T>(a.x * act::slope<ACT>(za.x), a.y * act::slope<ACT>(za.y), high.x, low.x);
        split_pair<T>(b.x * act::slope<ACT>(zb.x), b.y * act::slope<ACT>(zb.y), high.y, low.y);
    }
    return high;
}
// An infinity in the other operand meets the high part alone: times a low part of the other sign, or of zero, it would make the sum NaN.  `not_finite` is not zero where
// a 16-bit number of the words has all bits of its exponent set (those then carry into the sign's place); `finite_only` takes these numbers out.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w)
{
    constexpr uint32_t EXPONENT = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u, LOWEST = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
    return ((w & EXPONENT) + LOWEST) & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) { return w & ~((not_finite<T>(w) >> 15) * 0xFFFFu); }

__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
template <typename T>
constexpr int kind_of() { return std::is_same<T, __half>::value ? ASCB200_KIND_F16 : ASCB200_KIND_BF16; }

template <typename T, int ACT>
__device__ __forceinline__ void grad_rows_dx(const GradRowsArgs& p, float (*part)[kGradRows][kPartLd])
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int rank = blockIdx.x % p.splits, col0 = static_cast<int>(blockIdx.x / p.splits) * kGradStrip;
    const int chunks = (p.n + 15) / 16, per = (chunks + p.splits - 1) / p.splits;
    const int first = rank * per, last = min(chunks, first + per);
    const uint8_t* w = static_cast<const uint8_t*>(p.w);
    const long long ldw = p.ldw * 2;
    uint32_t acc[8][4];
    struct Piece {  // 16 rows x 64 columns of w, with the dz that meets them
        uint4 v[4];
        RawQuad dz[2];
    };
    auto load = [&](int ch, Piece& to) {
        const int row = ch * 16 + 4 * q, end = ch < last ? p.n : 0;
        const uint8_t* at = w + row * ldw;
#pragma unroll
        for (int j = 0; j < 4; ++j, at += ldw) {  // (what a piece holds from column k on belongs to no output; behind the last row it is not read)
            const int bytes = row + j < end ? (row + j < p.n - 1 ? (p.k + 7) / 8 * 16 : p.k * 2) : 0;
            to.v[j] = load_piece<true>(at, (col0 + 8 * g) * 2, bytes);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) to.dz[h] = load_dz<ACT>(p, end > 0 ? g + 8 * h : kGradRows, row);
    };
    // clean: the low parts meet finite weights alone
    auto add = [&](const Piece& from, auto clean) {
        uint2 first_low, second_low;  // rows g and g + 8
        const uint2 first_high = dz_of<T, ACT>(from.dz[0], first_low), second_high = dz_of<T, ACT>(from.dz[1], second_low);
        const uint32_t r0[4] = {from.v[0].x, from.v[0].y, from.v[0].z, from.v[0].w}, r1[4] = {from.v[1].x, from.v[1].y, from.v[1].z, from.v[1].w};
        const uint32_t r2[4] = {from.v[2].x, from.v[2].y, from.v[2].z, from.v[2].w}, r3[4] = {from.v[3].x, from.v[3].y, from.v[3].z, from.v[3].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t b0 = low_halves(r0[i], r1[i]), b1 = low_halves(r2[i], r3[i]), c0 = high_halves(r0[i], r1[i]), c1 = high_halves(r2[i], r3[i]);
            mma_16x8<kind_of<T>()>(acc[2 * i], first_high.x, second_high.x, first_high.y, second_high.y, b0, b1);
            mma_16x8<kind_of<T>()>(acc[2 * i + 1], first_high.x, second_high.x, first_high.y, second_high.y, c0, c1);
            if constexpr (!exact_dz<ACT>()) {
                if constexpr (clean.value) b0 = finite_only<T>(b0), b1 = finite_only<T>(b1), c0 = finite_only<T>(c0), c1 = finite_only<T>(c1);
                mma_16x8<kind_of<T>()>(acc[2 * i], first_low.x, second_low.x, first_low.y, second_low.y, b0, b1);
                mma_16x8<kind_of<T>()>(acc[2 * i + 1], first_low.x, second_low.x, first_low.y, second_low.y, c0, c1);
            }
        }
    };
    // Returns whether one of the thread's sums is not finite.
    auto strip = [&](auto clean) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0u;
        Piece even, odd;  // one is worked on while the other is on its way
        load(first + warp, even);
        for (int ch = first + warp; ch < last; ch += 2 * kGradWarps) {
            load(ch + kGradWarps, odd);
            add(even, clean);
            if (ch + kGradWarps >= last) break;
            load(ch + 2 * kGradWarps, even);
            add(odd, clean);
        }
        // place i * 8 + s holds column 8 s + i
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<float2*>(&part[warp][g + 8 * h][i * 8 + 2 * q]) = make_float2(__uint_as_float(acc[i][2 * h]), __uint_as_float(acc[i][2 * h + 1]));
        __syncthreads();
        bool bad = false;
        for (int i = threadIdx.x; i < kGradRows * kGradStrip; i += kGradThreads) {
            float* at = &part[0][i / kGradStrip][i % kGradStrip];
            float s = at[0];
#pragma unroll
            for (int v = 1; v < kGradWarps; ++v) s += at[v * kGradRows * kPartLd];
            at[0] = s;
            const int place = i % kGradStrip;
            bad |= !(fabsf(s) < __builtin_huge_valf()) && col0 + 8 * (place & 7) + (place >> 3) < p.k;
        }
        return bad;
    };
    // A sum that is not finite: an infinite weight may have met a low part.  The strip is then made once more, with the low parts meeting finite weights alone.
    // (Looking for infinities in every piece took up to 2 % of the whole.)
    const bool bad = strip(std::false_type());
    if constexpr (!exact_dz<ACT>())
        if (__syncthreads_or(bad)) strip(std::true_type());
    if (p.splits > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    const int share = (kGradRows * kGradStrip + p.splits - 1) / p.splits;
    for (int i = rank * share + threadIdx.x; i < min(kGradRows * kGradStrip, (rank + 1) * share); i += kGradThreads) {
        const int t = i / kGradStrip, c = i % kGradStrip, place = (c & 7) * 8 + (c >> 3);
        float s = 0.0f;
        if (p.splits > 1) {
            const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(&part[0][t][place]));
            for (int v = 0; v < p.splits; ++v) {
                uint32_t there;
                float f;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(v));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(there) : "memory");
                s += f;
            }
        } else {
            s = part[0][t][place];
        }
        if (t < p.m && col0 + c < p.k) static_cast<T*>(p.dx)[t * p.ld_dx + col0 + c] = rounded<T>(s);
    }
    if (p.splits > 1) {  // a block's sums stay until every block of the cluster has read them
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

constexpr int kALd = kGradTileRows + 8, kBLd = kGradTileCols + 2;  // words; so that a warp's reads fall into different banks
constexpr int kRunBytes = 256, kRunLd = kRunBytes + 16;            // of a row that a warp writes at once where rows do not start on 16 bytes
struct DwTile {
    uint32_t a[2][kGradRows / 2][kALd];  // rows 2 i and 2 i + 1 of dz, packed: high and low parts
    uint32_t b[kGradRows / 2][kBLd];  // and of x
    alignas(16) uint8_t out[kGradWarps][16][kRunLd];
};
// A warp writes 16 runs of `count` elements (of E bytes) from shared memory to rows `ld` elements apart, `rows` of which are there: a half warp per row, a
// lane per 16 bytes of the memory, the ends one by one.  (Element by element an SM's stores, each a partial 32-byte sector or three, took
// as long as the rest: 15 x 5312 x 1199 15.7 us for dw alone against 6.8 for 15 x 5312 x 1200.)
template <int E>
__device__ __forceinline__ void store_runs(uint8_t* to, long long ld, int rows, int count, const uint8_t (*from)[kRunLd], int lane)
{
    constexpr int N = 16 / E;  // elements per piece
#pragma unroll
    for (int h = 0; h < 16; h += 2) {
        const int r = h + (lane >> 4), l = lane & 15;
        if (r >= rows) continue;
        uint8_t* row = to + r * ld * E;
        const int head = min(count, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / E);
        const int pieces = (count - head) / N, tail = head + pieces * N;
        if (l < pieces) {
            const int e = (head + l * N) * E;  // its place in the run, a multiple of E
            const uint32_t* words = reinterpret_cast<const uint32_t*>(from[r]) + e / 4;
            uint32_t v[4];
            if (E == 4 || (e & 2) == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = words[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __byte_perm(words[j], words[j + 1], 0x5432);
            }
            *reinterpret_cast<uint4*>(row + e) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        const int single = l < 8 ? l : tail + l - 8;
        if (l < 8 ? single < head : single < count) {
            if constexpr (E == 4) reinterpret_cast<uint32_t*>(row)[single] = reinterpret_cast<const uint32_t*>(from[r])[single];
            else reinterpret_cast<uint16_t*>(row)[single] = reinterpret_cast<const uint16_t*>(from[r])[single];
        }
    }
}
// Two rows' quads -> four words, one per column.
__device__ __forceinline__ void put_pairs(uint32_t* to, uint2 a, uint2 b)
{
    to[0] = low_halves(a.x, b.x), to[1] = high_halves(a.x, b.x), to[2] = low_halves(a.y, b.y), to[3] = high_halves(a.y, b.y);
}
template <typename T, int ACT>
__device__ __forceinline__ void grad_rows_dw(const GradRowsArgs& p, DwTile& s)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    // A block has a run of tiles, along the columns first.  What a tile needs is requested while the one before it is made.
    const int across = (p.k + kGradTileCols - 1) / kGradTileCols, tiles = (p.n + kGradTileRows - 1) / kGradTileRows * across;
    const int block = blockIdx.x - p.dx_blocks;
    const int first = static_cast<int>(static_cast<long long>(block) * tiles / p.dw_blocks), last = static_cast<int>((block + 1ll) * tiles / p.dw_blocks);
    constexpr int kQuadsA = kGradTileRows / 4, kQuadsB = kGradTileCols / 4, kB = (kGradRows / 2) * kQuadsB / kGradThreads;
    const bool has_a = threadIdx.x < (kGradRows / 2) * kQuadsA;
    const int pair_a = threadIdx.x / kQuadsA, c_a = threadIdx.x % kQuadsA * 4;
    RawQuad raw_a[2];
    uint2 raw_b[kB][2];
    auto fetch = [&](int tile) {
        const int row0 = tile / across * kGradTileRows, col0 = tile % across * kGradTileCols;
        if (has_a) {
#pragma unroll
            for (int h = 0; h < 2; ++h) raw_a[h] = load_dz<ACT>(p, 2 * pair_a + h, row0 + c_a);
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = threadIdx.x + i * kGradThreads, pair = at / kQuadsB, c = at % kQuadsB * 4;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                raw_b[i][h] = 2 * pair + h < p.m ? load_quad(static_cast<const uint16_t*>(p.x) + (2 * pair + h) * p.ldx, col0 + c, p.k, true) : make_uint2(0u, 0u);
        }
    };
    if (first < last) fetch(first);
    for (int tile = first; tile < last; ++tile) {
        const int row0 = tile / across * kGradTileRows, col0 = tile % across * kGradTileCols;
        __syncthreads();  // the tile before has been read
        if (has_a) {
            uint2 low[2];
            const uint2 even = dz_of<T, ACT>(raw_a[0], low[0]), odd = dz_of<T, ACT>(raw_a[1], low[1]);
            put_pairs(&s.a[0][pair_a][c_a], even, odd);
            if constexpr (!exact_dz<ACT>()) put_pairs(&s.a[1][pair_a][c_a], low[0], low[1]);
        }
        uint32_t any = 0u;
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = threadIdx.x + i * kGradThreads;
            put_pairs(&s.b[at / kQuadsB][at % kQuadsB * 4], raw_b[i][0], raw_b[i][1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) any |= not_finite<T>(raw_b[i][h].x) | not_finite<T>(raw_b[i][h].y);
        }
        bool infinities = false;
        if constexpr (exact_dz<ACT>()) __syncthreads();
        else infinities = __syncthreads_or(any != 0u);
        if (tile + 1 < last) fetch(tile + 1);
        const int r = (warp & 3) * 16, half = (warp >> 2) * 128;
        const int run = p.dw_f32 ? 64 : 128;  // columns per run
        uint32_t a[2][4];
#pragma unroll
        for (int h = 0; h < (exact_dz<ACT>() ? 1 : 2); ++h) a[h][0] = s.a[h][q][r + g], a[h][1] = s.a[h][q][r + g + 8], a[h][2] = s.a[h][q + 4][r + g], a[h][3] = s.a[h][q + 4][r + g + 8];
        auto sets = [&](auto clean) {  // clean: the low parts meet finite numbers of x alone
#pragma unroll
            for (int set = 0; set < 4; ++set) {  // 32 columns: the lane gets eight of rows g and g + 8
                uint32_t d[4][4] = {};
                const int c = half + set * 32;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = c + 8 * (g >> 1) + 2 * i + (g & 1);
                    uint32_t b0 = s.b[q][at], b1 = s.b[q + 4][at];
                    mma_16x8<kind_of<T>()>(d[i], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
                    if constexpr (!exact_dz<ACT>()) {
                        if constexpr (clean.value) b0 = finite_only<T>(b0), b1 = finite_only<T>(b1);
                        mma_16x8<kind_of<T>()>(d[i], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = row0 + r + g + 8 * h, col = col0 + c + 8 * q;
                    uint8_t* staged = s.out[warp][g + 8 * h];
                    if (p.dw_f32) {
                        const uint4 v0 = make_uint4(d[0][2 * h], d[0][2 * h + 1], d[1][2 * h], d[1][2 * h + 1]), v1 = make_uint4(d[2][2 * h], d[2][2 * h + 1], d[3][2 * h], d[3][2 * h + 1]);
                        uint4* out = p.dw_vec ? reinterpret_cast<uint4*>(static_cast<float*>(p.dw) + row * p.ld_dw + col) : reinterpret_cast<uint4*>(staged + ((set & 1) * 32 + 8 * q) * 4);
                        if (!p.dw_vec || (row < p.n && col < p.k)) out[0] = v0, out[1] = v1;
                    } else {
                        uint32_t v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = pack_pair<T>(__uint_as_float(d[i][2 * h]), __uint_as_float(d[i][2 * h + 1]));
                        uint4* out = p.dw_vec ? reinterpret_cast<uint4*>(static_cast<T*>(p.dw) + row * p.ld_dw + col) : reinterpret_cast<uint4*>(staged + (set * 32 + 8 * q) * 2);
                        if (!p.dw_vec || (row < p.n && col < p.k)) *out = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                if (!p.dw_vec && (set == 3 || (p.dw_f32 && set == 1))) {  // a run of 256 bytes per row is together
                    __syncwarp();
                    const int col = col0 + half + (p.dw_f32 ? (set >> 1) * 64 : 0), count = min(run, p.k - col), rows = min(16, p.n - row0 - r);
                    const long long at = static_cast<long long>(row0 + r) * p.ld_dw + col;
                    if (count > 0 && rows > 0) {
                        if (p.dw_f32) store_runs<4>(static_cast<uint8_t*>(p.dw) + at * 4, p.ld_dw, rows, count, s.out[warp], lane);
                        else store_runs<2>(static_cast<uint8_t*>(p.dw) + at * 2, p.ld_dw, rows, count, s.out[warp], lane);
                    }
                    __syncwarp();
                }
            }
        };
        if (infinities) sets(std::true_type());
        else sets(std::false_type());
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kGradThreads, 2)
grad_rows_kernel(const GradRowsArgs p)
{
    __shared__ alignas(16) union {
        float part[kGradWarps][kGradRows][kPartLd];
        DwTile tile;
    } s;
    const int block = blockIdx.x;
    if (block < p.dx_blocks) {  // while the kernel before this one drains, ask L2 for the first pieces of w (hints only)
        const int chunks = (p.n + 15) / 16, per = (chunks + p.splits - 1) / p.splits;
        const int row = (block % p.splits) * per * 16 + threadIdx.x;
        if (row < p.n) asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(p.w) + (row * p.ldw + block / p.splits * kGradStrip) * 2));
    }
    grid_dependency_wait();
    if (block < p.dx_blocks) {
        grad_rows_dx<T, ACT>(p, s.part);
    } else if (block < p.dx_blocks + p.dw_blocks) {
        grad_rows_dw<T, ACT>(p, s.tile);
    } else {
        const int c = (block - p.dx_blocks - p.dw_blocks) * kGradThreads + threadIdx.x;
        if (!p.dbias || c >= p.n) return;
        float v = 0.0f;
#pragma unroll
        for (int t = 0; t < kGradRows; ++t) {
            if (t >= p.m) break;
            float f = as_f32(static_cast<const T*>(p.dy)[t * p.ld_dy + c]);
            if constexpr (ACT != ASCB200_ACT_NONE) f *= act::slope<ACT>(as_f32(static_cast<const T*>(p.z)[t * p.ldz + c]));
            v += f;
        }
        if (p.dbias_f32) static_cast<float*>(p.dbias)[c] = v;
        else static_cast<T*>(p.dbias)[c] = rounded<T>(v);
    }
}

template <typename T>
int launch_grad_rows(GradRowsArgs p, int act, int sms, cudaStream_t st)
{
    const int strips = (p.k + kGradStrip - 1) / kGradStrip, chunks = (p.n + 15) / 16;
    // w's rows are split while two blocks per SM hold all strips' parts at once and every warp still has a piece.
    p.splits = p.dx ? std::max(1, std::min({8, 2 * sms / strips, chunks / kGradWarps})) : 1;
    p.dx_blocks = p.dx ? strips * p.splits : 0;
    const long long tiles = p.dw ? static_cast<long long>((p.n + kGradTileRows - 1) / kGradTileRows) * ((p.k + kGradTileCols - 1) / kGradTileCols) : 0;
    p.dw_blocks = static_cast<int>(std::min(tiles, (p.dx ? 4ll : 2ll) * sms));  // (behind dx shorter runs fill the SMs more evenly: 16 x 4096 x 11008 50 against 60 us)
    int blocks = p.dx_blocks + p.dw_blocks + (p.dbias ? (p.n + kGradThreads - 1) / kGradThreads : 0);
    blocks = (blocks + p.splits - 1) / p.splits * p.splits;
    switch (act) {
#define ASCB200_GRAD_ROWS(A) case A: ASCB200_CUDA(launch_pdl_cluster(grad_rows_kernel<T, A>, blocks, kGradThreads, 0, st, p.splits, p)); return ASCB200_OK;
        ASCB200_GRAD_ROWS(ASCB200_ACT_FASTER_GELU)
        ASCB200_GRAD_ROWS(ASCB200_ACT_RELU)
        ASCB200_GRAD_ROWS(ASCB200_ACT_GELU)
        ASCB200_GRAD_ROWS(ASCB200_ACT_GELU_TANH)
        ASCB200_GRAD_ROWS(ASCB200_ACT_SILU)
        default: ASCB200_CUDA(launch_pdl_cluster(grad_rows_kernel<T, ASCB200_ACT_NONE>, blocks, kGradThreads, 0, st, p.splits, p)); return ASCB200_OK;
#undef ASCB200_GRAD_ROWS
    }
}

constexpr int kActGradBlocks = 592;  // blocks to aim for: four per SM
int act_grad_row_blocks(int m, int n)
{
    const int cols = (n + 255) / 256;
    if (m <= 32) return 1;  // a launch less (us, fp16 silu with dbias: 17 x 128 x 335 10.6 -> 9.8, 20 x 4096 x 1024 20.9 -> 20.2; 64 x 11008 x 1024 would take 34.0 for 31.6)
    return static_cast<int>(std::min<long long>((m + 7ll) / 8, std::max(1, std::min(296, kActGradBlocks / cols))));
}
size_t dz_bytes(int m, int n) { return (static_cast<size_t>(m) * ((static_cast<size_t>(n) + 7) / 8 * 8) * 2 + 255) / 256 * 256; }
size_t linear_grad_workspace(int m, int n)
{
    return m <= 0 || n <= 0 ? 0 : dz_bytes(m, n) + static_cast<size_t>(act_grad_row_blocks(m, n)) * n * sizeof(float);
}

int run_linear_grad(const ascb200_linear_grad_desc* desc, cudaStream_t stream)
{
    DeviceState* state = current_state();
    if (!state) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_linear_grad_desc d = *desc;
    if (d.m < 0 || d.n <= 0 || d.k <= 0 || (d.trans_w != 0 && d.trans_w != 1)) return ASCB200_EINVAL;
    if (d.act < ASCB200_ACT_NONE || d.act > ASCB200_ACT_SILU) return ASCB200_EINVAL;
    if (d.kind != ASCB200_KIND_F16 && d.kind != ASCB200_KIND_BF16) return ASCB200_EUNSUPPORTED;
    const int own = d.kind == ASCB200_KIND_F16 ? ASCB200_F16 : ASCB200_BF16;
    if (d.dw_dev && d.dw_dtype != own && d.dw_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    if (d.dbias_dev && d.dbias_dtype != own && d.dbias_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    const int w_cols = d.trans_w ? d.k : d.n, w_rows = d.trans_w ? d.n : d.k;
    if (d.ld_dy == 0) d.ld_dy = d.n;
    if (d.ldz == 0) d.ldz = d.n;
    if (d.ldx == 0) d.ldx = d.k;
    if (d.ldw == 0) d.ldw = w_cols;
    if (d.ld_dx == 0) d.ld_dx = d.k;
    if (d.ld_dw == 0) d.ld_dw = w_cols;
    if (d.ld_dy < d.n || d.ldz < d.n || d.ldx < d.k || d.ldw < w_cols || d.ld_dx < d.k || d.ld_dw < w_cols) return ASCB200_EINVAL;
    const int dwsz = float_bytes(d.dw_dtype), dbsz = float_bytes(d.dbias_dtype);
    if ((d.dw_dev && !element_aligned(d.dw_dev, dwsz)) || (d.dbias_dev && !element_aligned(d.dbias_dev, dbsz))) return ASCB200_EALIGN;
    if (d.m == 0) {  // no rows: dw and dbias are sums of nothing
        if (d.dw_dev) ASCB200_CUDA(cudaMemset2DAsync(d.dw_dev, static_cast<size_t>(d.ld_dw) * dwsz, 0, static_cast<size_t>(w_cols) * dwsz, w_rows, stream));
        if (d.dbias_dev) ASCB200_CUDA(cudaMemsetAsync(d.dbias_dev, 0, static_cast<size_t>(d.n) * dbsz, stream));
        return ASCB200_OK;
    }
    if (!d.dy_dev || (d.act != ASCB200_ACT_NONE && !d.z_dev) || (d.dx_dev && !d.w_dev) || (d.dw_dev && !d.x_dev)) return ASCB200_EINVAL;
    if (!element_aligned(d.dy_dev, 2) || !element_aligned(d.z_dev, 2) || !element_aligned(d.dx_dev, 2)) return ASCB200_EALIGN;
    if ((d.dx_dev && !operand_aligned(d.w_dev, d.ldw, 2)) || (d.dw_dev && !operand_aligned(d.x_dev, d.ldx, 2))) return ASCB200_EALIGN;

    // A product whose rows do not start on 16 bytes is stored by the linear build's output stage, which writes runs of a row through shared
    // memory (gradients of 777 x 1000 x 515 fp16: 39.1 us in all with the plain build's element stores, 21.7 so).
    // Products of few tiles leave most SMs idle, and each has its latency: then both run side by side (us, all of the gradient, m x n x k: 777 x 1000 x 515
    // 20.9 -> 14.1, 85 x 128 x 100 10.9 -> 7.6, 420 x 8256 x 755 44.6 -> 38.9, 35 x 5417 x 2742 41.3 -> 37.2; nothing for 2048 x 2048 x 2048, and
    // 4096 x 4096 x 1024 76 -> 81: there the plain build and the order of two full waves are better).
    auto tiles = [](long long rows, long long cols) { return (rows + 127) / 128 * ((cols + 127) / 128); };
    const bool together = d.dx_dev && d.dw_dev && tiles(d.m, d.k) + tiles(w_rows, w_cols) <= 8ll * state->sm_count;
    gemm::LinearArgs nothing = {nullptr, 0, ASCB200_ACT_NONE, nullptr, 0};
    auto product = [&](const ascb200_gemm_desc& q, int order) {
        const bool aligned = aligned_to(q.c_dev, 16) && (q.ldc * float_bytes(q.c_dtype)) % 16 == 0;
        nothing.order = together ? order : 0;
        return gemm::run_gemm(&q, nullptr, 0, stream, nullptr, aligned && !together ? nullptr : &nothing);
    };
    const bool products = d.dx_dev || d.dw_dev;
    // dy itself is the operand where there is no activation and it can be one
    const bool make_dz = products && (d.act != ASCB200_ACT_NONE || !operand_aligned(d.dy_dev, d.ld_dy, 2));
    const void* dz = d.dy_dev;
    int64_t ld_dz = d.ld_dy;
    if (make_dz || d.dbias_dev) {
        if (!d.workspace_dev || d.workspace_bytes < linear_grad_workspace(d.m, d.n)) return ASCB200_EINVAL;
        if (!aligned_to(d.workspace_dev, 16)) return ASCB200_EALIGN;
    }
    if (d.m <= kGradRows && d.trans_w && products && d.k < (1 << 30)) {
        GradRowsArgs p = {};
        p.dy = d.dy_dev, p.z = d.z_dev, p.x = d.x_dev, p.w = d.w_dev, p.dx = d.dx_dev, p.dw = d.dw_dev, p.dbias = d.dbias_dev;
        p.ld_dy = d.ld_dy, p.ldz = d.ldz, p.ldx = d.ldx, p.ldw = d.ldw, p.ld_dx = d.ld_dx, p.ld_dw = d.ld_dw, p.m = d.m, p.n = d.n, p.k = d.k;
        p.dw_f32 = d.dw_dtype == ASCB200_F32, p.dbias_f32 = d.dbias_dtype == ASCB200_F32;
        p.quads = aligned_to(d.dy_dev, 8) && d.ld_dy % 4 == 0 && (d.act == ASCB200_ACT_NONE || (aligned_to(d.z_dev, 8) && d.ldz % 4 == 0));
        p.dw_vec = d.k % 8 == 0 && aligned_to(d.dw_dev, 16) && (d.ld_dw * dwsz) % 16 == 0;
        return d.kind == ASCB200_KIND_F16 ? launch_grad_rows<__half>(p, d.act, state->sm_count, stream) : launch_grad_rows<__nv_bfloat16>(p, d.act, state->sm_count, stream);
    }
    if (make_dz || d.dbias_dev) {
        ActGradArgs p = {};
        p.dy = d.dy_dev, p.z = d.z_dev, p.ld_dy = d.ld_dy, p.ldz = d.ldz, p.m = d.m, p.n = d.n;
        if (make_dz) {
            dz = p.dz = d.workspace_dev;
            ld_dz = p.ld_dz = (static_cast<int64_t>(d.n) + 7) / 8 * 8;
        }
        p.dbias = d.dbias_dev, p.dbias_f32 = d.dbias_dtype == ASCB200_F32;
        if (d.dbias_dev) p.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(d.workspace_dev) + dz_bytes(d.m, d.n));
        const bool vec = d.n % 8 == 0 && operand_aligned(d.dy_dev, d.ld_dy, 2) && (d.act == ASCB200_ACT_NONE || operand_aligned(d.z_dev, d.ldz, 2));
        const int rows = act_grad_row_blocks(d.m, d.n);
        const dim3 grid((d.n + 255) / 256, rows);
        const int rc = d.kind == ASCB200_KIND_F16 ? launch_act_grad<__half>(p, d.act, vec, grid, stream) : launch_act_grad<__nv_bfloat16>(p, d.act, vec, grid, stream);
        if (rc != ASCB200_OK) return rc;
        if (d.dbias_dev && rows > 1) {
            const int rc2 = sum_partials(p.partial, d.dbias_dev, d.dbias_dtype, rows, d.n, stream);
            if (rc2 != ASCB200_OK) return rc2;
        }
    }
    if (d.dx_dev) {  // [m, k] = dz [m, n] * w
        ascb200_gemm_desc q = {};
        q.kind = d.kind, q.m = d.m, q.n = d.k, q.k = d.n;
        q.a_dev = dz, q.lda = ld_dz, q.b_dev = d.w_dev, q.ldb = d.ldw, q.trans_b = !d.trans_w;
        q.c_dev = d.dx_dev, q.ldc = d.ld_dx, q.c_dtype = own;
        const int rc = product(q, gemm::kFirstOfTwo);
        if (rc != ASCB200_OK) return rc;
    }
    if (d.dw_dev) {  // [n, k] = dz^T x, or [k, n] = x^T dz
        ascb200_gemm_desc q = {};
        q.kind = d.kind, q.m = w_rows, q.n = w_cols, q.k = d.m, q.trans_a = 1;
        q.a_dev = d.trans_w ? dz : d.x_dev, q.lda = d.trans_w ? ld_dz : d.ldx;
        q.b_dev = d.trans_w ? d.x_dev : dz, q.ldb = d.trans_w ? d.ldx : ld_dz;
        q.c_dev = d.dw_dev, q.ldc = d.ld_dw, q.c_dtype = d.dw_dtype;
        const int rc = product(q, gemm::kSecondOfTwo);
        if (rc != ASCB200_OK) return rc;
    }
    return ASCB200_OK;
}

}  // namespace
}  // namespace ascb200

extern "C" {

int ascb200_linear(const ascb200_linear_desc* desc, void* stream) { return ascb200::run_linear(desc, static_cast<cudaStream_t>(stream)); }

size_t ascb200_linear_grad_workspace_bytes(int32_t m, int32_t n) { return ascb200::linear_grad_workspace(m, n); }

int ascb200_linear_grad(const ascb200_linear_grad_desc* desc, void* stream) { return ascb200::run_linear_grad(desc, static_cast<cudaStream_t>(stream)); }

}  // extern "C"
