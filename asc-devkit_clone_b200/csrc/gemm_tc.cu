// Host side of the tensor-core GEMM (kernels: gemm_kernels.cuh): argument checks, tensor maps, tile choice, the re-tiling of MX
// scale factors, and the C entry points of the matrix products.
#include <algorithm>
#include <cstring>
#include <mutex>

#include "gemm_host.cuh"
#include "gemm_linear.cuh"

namespace ascb200 {
namespace gemm {
namespace {

// Re-tiles MX scale factors [rows, ks] (row-major bytes) into 512-byte chunks: chunk (rb, kc) holds
// the scales of rows rb*128 .. +127 and K-blocks kc*4 .. +3 at byte (r%32)*16 + (r/32)*4 + (ks%4),
// the order tcgen05.cp (32x128b, warpx4) expects.  Missing rows / K-blocks are filled with 127 (1.0).
// One launch covers both operands: blocks [0, rb_a * kc_tiles) re-tile A, the rest B.  A block moves
// 128 rows x 8 chunks through shared memory so that rows are read as whole sectors and chunks written as whole lines.
// `paired` bit 0 / 1: the source of A / B is stored [ks / 2][rows][2] instead (the two scales of a 64-element K step side
// by side, rows next): the order the reference keeps a transposed scaleA and a non-transposed scaleB in
// (examples/.../00_matmul/matmul_mx/scripts/gen_data.py: reshape(sk / 2, 2, n).transpose(0, 2, 1)).
__global__ void __launch_bounds__(256)
retile_scales_kernel(const uint8_t* __restrict__ src_a, uint32_t* __restrict__ dst_a, int rows_a, int rb_a, const uint8_t* __restrict__ src_b,
                     uint32_t* __restrict__ dst_b, int rows_b, int ks, int kc_count, int kc_tiles, int paired)
{
    constexpr int CH = 8;  // chunks per block: 32 bytes of every row, four words per thread, all loads issued before any is used
    __shared__ uint32_t tile[128][CH + 1];  // [position inside a chunk][chunk]
    grid_dependency_wait();
    int blk = blockIdx.x;
    const bool is_a = blk < rb_a * kc_tiles;
    if (!is_a) blk -= rb_a * kc_tiles;
    const uint8_t* src = is_a ? src_a : src_b;
    uint32_t* dst = is_a ? dst_a : dst_b;
    const int rows = is_a ? rows_a : rows_b;
    const int rb = blk / kc_tiles, kc0 = (blk % kc_tiles) * CH;
    const bool pair_src = ((paired >> (is_a ? 0 : 1)) & 1) != 0;
    const bool words = !pair_src && (ks & 3) == 0 && (reinterpret_cast<uintptr_t>(src) & 3) == 0;
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int idx = threadIdx.x + u * 256;
        // plain source: consecutive threads read along a row; paired source: consecutive threads read consecutive rows
        const int rl = pair_src ? idx % 128 : idx / CH, j = pair_src ? idx / 128 : idx % CH;
        const int r = rb * 128 + rl, k = (kc0 + j) * 4;
        if (pair_src) {
            w[u] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                w[u] |= ((r < rows && k + b < ks) ? static_cast<uint32_t>(src[(static_cast<size_t>((k + b) >> 1) * rows + r) * 2 + ((k + b) & 1)]) : 127u)
                        << (8 * b);
        } else if (r < rows && k + 3 < ks && words) {
            w[u] = __ldg(reinterpret_cast<const uint32_t*>(src + static_cast<size_t>(r) * ks + k));
        } else {
            w[u] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) w[u] |= ((r < rows && k + b < ks) ? static_cast<uint32_t>(src[static_cast<size_t>(r) * ks + k + b]) : 127u) << (8 * b);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int idx = threadIdx.x + u * 256;
        const int rl = pair_src ? idx % 128 : idx / CH, j = pair_src ? idx / 128 : idx % CH;
        tile[(rl & 31) * 4 + (rl >> 5)][j] = w[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int idx = threadIdx.x + u * 256;
        const int j = idx >> 7, pos = idx & 127;
        if (kc0 + j < kc_count) dst[(static_cast<size_t>(rb) * kc_count + kc0 + j) * 128 + pos] = tile[pos][j];
    }
}

// ---- host side --------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(f);
        else
            (void)cudaGetLastError();
    });
    return fn;
}

// rank-3 map over [d2][d1][d0] (d0 contiguous), box {b0, b1, 1}, 128-byte swizzle, zero fill out of bounds.
int make_map(CUtensorMap* map, CUtensorMapDataType dt, int esz, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t stride1_elems,
             uint64_t stride2_elems, uint32_t b0, uint32_t b1)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) return ASCB200_ECUDA;
    cuuint64_t dims[3] = {d0, d1, d2};
    cuuint64_t strides[2] = {stride1_elems * esz, stride2_elems * esz};
    cuuint32_t box[3] = {b0, b1, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    if (!aligned_to(base, 16) || strides[0] % 16 != 0 || strides[1] % 16 != 0) return ASCB200_EALIGN;
    CUresult r = fn(map, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ASCB200_OK : ASCB200_ECUDA;
}

// rank-2 map over re-tiled scales: `chunks` rows of 128 x u32 (512 bytes), box = box_rows rows, no swizzle.
int make_sf_map(CUtensorMap* map, const void* base, uint64_t chunks, uint32_t box_rows)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) return ASCB200_ECUDA;
    cuuint64_t dims[2] = {128, chunks};
    cuuint64_t strides[1] = {SF_CHUNK_BYTES};
    cuuint32_t box[2] = {128, box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? ASCB200_OK : ASCB200_ECUDA;
}

int out_bytes(int dt) { return (dt == OUT_S8 || dt == OUT_E4M3 || dt == OUT_E5M2) ? 1 : (dt == OUT_F16 || dt == OUT_BF16) ? 2 : 4; }

// rank-2 map over an output [rows][cols] of 1- or 2-byte elements, box 32 x 32, swizzle = bytes of one box row.
// Returns false when the tensor cannot be described (alignment): the kernel then stores from registers.
bool make_out_map(CUtensorMap* map, int dtype, const void* base, uint64_t cols, uint64_t rows, uint64_t ld_elems)
{
    const int esz = out_bytes(dtype);
    // plain stores move bits; a reducing store (atomic add) needs the arithmetic type
    const CUtensorMapDataType mdt = dtype == OUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : dtype == OUT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                                                           : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    EncodeTiledFn fn = encode_fn();
    if (!fn || (esz != 1 && esz != 2) || !aligned_to(base, 16) || (ld_elems * esz) % 16 != 0 || cols == 0 || rows == 0) return false;
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {ld_elems * esz};
    cuuint32_t box[2] = {32, 32};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, mdt, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, esz == 1 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS;
}

// Split K over a cluster (single-CTA kernel): 4 or 2 CTAs per tile, or 0.  Time of a small problem ~ 5 us fixed + 0.21 us per K
// block of the longest CTA + 1.5 / 2.8 us for the exchange with 2 / 4 CTAs (fitted to fp16 512 x 512 x K: K = 1024, 16 blocks,
// 8.3 -> 8.6 / 9.1 us with 2 / 4 CTAs; K = 2048: 11.9 -> 10.4 / 10.2; K = 4096: 19.5 -> 14.5 / 12.5; and 128 x 1024 x 8192: 33.8 ->
// 21.7 / 15.7).  Every cluster needs a tile of its own, every CTA a K block, and the other CTAs' accumulators (block_n x 512 bytes
// each) must fit the leader's operand ring (about 192 KB).  `gain`: estimated time relative to no split.
int pick_split_k(long long tiles, int num_k_blocks, int block_n, int sm_count, double* gain = nullptr)
{
    const double fixed = 5.0, per_block = 0.21, exchange[5] = {0.0, 0.0, 1.5, 0.0, 2.8};
    const double base = fixed + per_block * num_k_blocks;
    int best = 0;
    double best_t = base;
    for (int sk = 2; sk <= 4; sk <<= 1) {
        if (tiles * sk > sm_count || num_k_blocks < 2 * sk) continue;
        if (static_cast<long long>(sk - 1) * block_n * 512 > 192 * 1024) continue;
        const double t = fixed + per_block * ((num_k_blocks + sk - 1) / sk) + exchange[sk];
        if (t < 0.97 * best_t) {
            best_t = t;
            best = sk;
        }
    }
    if (gain) *gain = best_t / base;
    return best;
}

bool is_mxfp8(int kind) { return kind == ASCB200_KIND_MXFP8_E4M3 || kind == ASCB200_KIND_MXFP8_E5M2; }
bool is_mx(int kind) { return kind == ASCB200_KIND_MXFP4 || is_mxfp8(kind); }
int elem_bits(int kind) { return kind == ASCB200_KIND_MXFP4 ? 4 : (kind == ASCB200_KIND_S8 || is_mxfp8(kind)) ? 8 : 16; }

}  // namespace

int run_gemm(const ascb200_gemm_desc* d, const int64_t* group_counts, int groups, cudaStream_t stream, const FixedResources* fixed, const LinearArgs* linear)
{
    DeviceState* st = fixed ? nullptr : current_state();
    if (!fixed && !st) return ASCB200_ENODEV;
    const int sm_count = fixed ? fixed->sm_count : st->sm_count;
    if (!d) return ASCB200_EINVAL;
    if (d->m < 0 || d->n < 0 || d->k < 0) return ASCB200_EINVAL;
    if (d->m == 0 || d->n == 0) return ASCB200_OK;
    if (!d->a_dev || !d->b_dev || !d->c_dev || d->k == 0) return ASCB200_EINVAL;
    if (d->reserved[0] != 0) return ASCB200_EINVAL;
    if (d->c_layout < ASCB200_C_ROW_MAJOR || d->c_layout > ASCB200_C_NZ) return ASCB200_EINVAL;
    if (d->c_layout != ASCB200_C_ROW_MAJOR && (d->atomic || d->c2_dev || groups > 0)) return ASCB200_EUNSUPPORTED;
    if (d->scale_flags & ~(ASCB200_SCALE_A_PREPACKED | ASCB200_SCALE_B_PREPACKED | ASCB200_SCALE_A_PAIRED | ASCB200_SCALE_B_PAIRED)) return ASCB200_EINVAL;
    const int kind = d->kind;
    if (kind < ASCB200_KIND_F16 || kind > ASCB200_KIND_MXFP8_E5M2) return ASCB200_EINVAL;
    const bool acc_int = kind == ASCB200_KIND_S8;
    const bool grouped = groups > 0;
    if (grouped && (groups > MAX_GROUPS)) return ASCB200_ETOOBIG;
    if (grouped && (!group_counts || kind != ASCB200_KIND_S8 || d->epilogue != ASCB200_EPI_DEQUANT_TOKEN_CHANNEL || d->trans_a)) return ASCB200_EUNSUPPORTED;

    // ---- epilogue validation ----
    EpiParams e = {};
    e.c = d->c_dev;
    e.layout = d->c_layout;
    e.ldc = d->ldc ? d->ldc : (d->c_layout == ASCB200_C_ROW_MAJOR ? d->n : d->m);
    e.c_dtype = d->c_dtype;
    e.mode = d->epilogue;
    e.relu = d->relu;
    e.act = d->act;
    e.bias = d->bias_dev;
    e.tok = d->tok_scale_dev;
    e.ch = d->ch_scale_dev;
    e.quant = reinterpret_cast<const unsigned long long*>(d->quant_dev);
    e.quant_scalar = d->quant_scalar;
    if (e.ldc < (e.layout == ASCB200_C_ROW_MAJOR ? d->n : d->m)) return ASCB200_EINVAL;
    switch (d->epilogue) {
        case ASCB200_EPI_CAST:
            if (acc_int ? d->c_dtype != OUT_S32 : !(d->c_dtype == OUT_F32 || d->c_dtype == OUT_F16 || d->c_dtype == OUT_BF16)) return ASCB200_EUNSUPPORTED;
            break;
        case ASCB200_EPI_FIXPIPE_QUANT:
            if (acc_int ? !(d->c_dtype == OUT_F16 || d->c_dtype == OUT_S8 || d->c_dtype == OUT_BF16)
                        : !(d->c_dtype == OUT_S8 || d->c_dtype == OUT_F16 || d->c_dtype == OUT_BF16 || d->c_dtype == OUT_F32 || d->c_dtype == OUT_E4M3 ||
                            d->c_dtype == OUT_E5M2))
                return ASCB200_EUNSUPPORTED;
            break;
        case ASCB200_EPI_DEQUANT_TOKEN_CHANNEL:
            if (!acc_int || !d->ch_scale_dev) return ASCB200_EINVAL;
            if (!(d->c_dtype == OUT_F32 || d->c_dtype == OUT_F16 || d->c_dtype == OUT_BF16)) return ASCB200_EUNSUPPORTED;
            break;
        default: return ASCB200_EINVAL;
    }
    if (d->act != 0 && !(d->act == 1 && d->epilogue == ASCB200_EPI_DEQUANT_TOKEN_CHANNEL)) return ASCB200_EUNSUPPORTED;
    if (d->c2_dev) {
        if (acc_int || !(d->c2_dtype == OUT_F32 || d->c2_dtype == OUT_F16 || d->c2_dtype == OUT_BF16)) return ASCB200_EUNSUPPORTED;
        e.c2 = d->c2_dev;
        e.ldc2 = d->ldc2 ? d->ldc2 : d->n;
        e.c2_dtype = d->c2_dtype;
        if (e.ldc2 < d->n) return ASCB200_EINVAL;
        e.vec_c2 = aligned_to(e.c2, 16) && (e.ldc2 * out_bytes(e.c2_dtype)) % 16 == 0;
    }
    e.vec_c = aligned_to(e.c, 16) && (e.ldc * out_bytes(e.c_dtype)) % 16 == 0;
    // 1- and 2-byte outputs leave through shared memory and bulk tensor stores when their layout allows a tensor map
    OutMaps outs;
    std::memset(&outs, 0, sizeof(outs));
    const bool no_tma_store = getenv("ASCB200_NO_TMA_STORE") && getenv("ASCB200_NO_TMA_STORE")[0] == '1';
    e.tma_c = !no_tma_store && e.layout == ASCB200_C_ROW_MAJOR && make_out_map(&outs.c, e.c_dtype, e.c, d->n, d->m, e.ldc);
    e.tma_c2 = !no_tma_store && e.c2 && make_out_map(&outs.c2, e.c2_dtype, e.c2, d->n, d->m, e.ldc2);
    e.atomic = d->atomic;
    if (d->atomic < 0 || d->atomic > 3) return ASCB200_EUNSUPPORTED;                         // enAtomic: 0 off, 1 add, 2 max, 3 min
    if (d->atomic && out_bytes(e.c_dtype) == 1) return ASCB200_EUNSUPPORTED;                 // no 8-bit atomics
    if (d->atomic && out_bytes(e.c_dtype) == 2 && (reinterpret_cast<uintptr_t>(e.c) & 1)) return ASCB200_EALIGN;

    // ---- operands ----
    const int bits = elem_bits(kind);
    const int k = d->k, m = d->m, n = d->n;
    if (is_mx(kind)) {
        // K a multiple of 64 like the reference's MmadMx
        if (k % 64 != 0) return ASCB200_EINVAL;
        if (!d->scale_a_dev || !d->scale_b_dev) return ASCB200_EINVAL;
    }
    if (kind == ASCB200_KIND_MXFP4) {
        if (d->trans_a || !d->trans_b) {
            // The tensor core takes fp4 operands K-major only.  An operand stored the other way round ([K, M] / the reference's
            // ND [K, N], two M- / N-neighbours per byte) is transposed into this stream's scratch first, then the call
            // proceeds on the copies; the scale scratch follows them in the same block.
            if (fixed) return ASCB200_EUNSUPPORTED;   // the allocation-free entry point has no room for operand copies
            if ((d->trans_a && ((m & 1) || (d->lda && d->lda != m))) || (!d->trans_b && ((n & 1) || (d->ldb && d->ldb != n)))) return ASCB200_EUNSUPPORTED;
            auto round256 = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
            const size_t bytes_ta = d->trans_a ? round256(static_cast<size_t>(m) * k / 2) : 0;
            const size_t bytes_tb = !d->trans_b ? round256(static_cast<size_t>(n) * k / 2) : 0;
            const size_t kc2 = 2 * static_cast<size_t>((k + 255) / 256);
            const size_t bytes_sf = (static_cast<size_t>((m + 127) / 128) + (n + 127) / 128 + kSfPadBlocks) * kc2 * SF_CHUNK_BYTES;
            void* ptr = nullptr;
            int rc0 = stream_scratch(st, bytes_ta + bytes_tb + bytes_sf, stream, &ptr);
            if (rc0 != ASCB200_OK) return rc0;
            uint8_t* base = static_cast<uint8_t*>(ptr);
            ascb200_gemm_desc d2 = *d;
            if (d->trans_a) {
                rc0 = fp4_transpose(d->a_dev, base, k, m, stream);
                if (rc0 != ASCB200_OK) return rc0;
                d2.a_dev = base;
                d2.trans_a = 0;
                d2.lda = 0;
            }
            if (!d->trans_b) {
                rc0 = fp4_transpose(d->b_dev, base + bytes_ta, k, n, stream);
                if (rc0 != ASCB200_OK) return rc0;
                d2.b_dev = base + bytes_ta;
                d2.trans_b = 1;
                d2.ldb = 0;
            }
            FixedResources sub = {st->status_dev, base + bytes_ta + bytes_tb, bytes_sf, st->sm_count, st->l2_bytes};
            return run_gemm(&d2, nullptr, 0, stream, &sub);
        }
    }
    const int64_t lda = d->lda ? d->lda : (d->trans_a ? m : k);
    const int64_t ldb = d->ldb ? d->ldb : (d->trans_b ? k : n);
    const int esz = bits == 16 ? 2 : 1;                // bytes per tensor-map element
    const int epb = bits == 4 ? 2 : 1;                 // logical elements per tensor-map element
    const CUtensorMapDataType dt = kind == ASCB200_KIND_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                 : kind == ASCB200_KIND_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint32_t row_elems = ROW_BYTES / esz;        // tensor-map elements per 128-byte row
    const int block_k = bits == 16 ? 64 : bits == 8 ? 128 : 256;

    // Tile choice: estimated time = waves x tile work / efficiency of that tile shape (wider tiles read less shared
    // memory and L2 per MAC; measured on 4096 x 4096 x 11008 int8: pair 256x256 1.0, single 128x256 0.88, 128x128 0.75,
    // 128x64 0.5).  Small problems and thin N-slabs get narrower tiles so that the last wave is not mostly idle.
    const int pair_clusters = sm_count / 2;
    const bool pair_possible = !(getenv("ASCB200_NO_PAIR") && getenv("ASCB200_NO_PAIR")[0] == '1');
    // Grouped problems on CTA pairs: full 256-row blocks of a group run like a plain GEMM; the group's last, partial block
    // is multiplied with the operand roles swapped (the pair's 256 weight rows become the M side of the instruction, the
    // block's rows, rounded up to 16, its N side), so that at most 15 rows per group are multiplied in vain.  Without the
    // swap a group's last 256-row tile is half empty on average, and under the board's power cap the wasted MMAs cost as
    // much time as useful ones (64 groups of 512 rows on average: masked pairs 490 us, single-CTA tiles 406-475 us).
    const bool group_swap_ok = grouped && !(getenv("ASCB200_NO_GROUP_SWAP") && getenv("ASCB200_NO_GROUP_SWAP")[0] == '1');
    const bool pair_allowed = pair_possible && (!grouped || group_swap_ok || m / groups >= 16 * BLOCK_M);
    const int wide = is_mx(kind) ? 192 : 256;   // block-scaled kinds at 256 columns cannot double-buffer their accumulators in TMEM
    int block_n = 64;
    bool use_pair = false;
    {
        const long long m_tiles = grouped ? (m + BLOCK_M - 1) / BLOCK_M + groups : (m + BLOCK_M - 1) / BLOCK_M;
        double best = -1.0;
        struct Cand { int bn; bool pair; double eff; };
        Cand cands[20];
        int num_cands = 0;
        cands[num_cands++] = {wide, true, 1.0};
        if (!is_mx(kind) && d->trans_b && !(grouped && group_swap_ok)) {
            // CTA-pair tiles of any width that is a multiple of 16: a narrower tile re-reads A more often per column
            // (128 columns measured at 0.75 of the full width's rate), but may fill the last wave far better
            for (int bn = 240; bn >= 64; bn -= 16) cands[num_cands++] = {bn, true, 1.0 / (1.0 + 0.33 * (256.0 / bn - 1.0))};
        }
        cands[num_cands++] = {wide, false, 0.88};
        cands[num_cands++] = {128, false, 0.75};
        cands[num_cands++] = {64, false, 0.5};
        for (int ci = 0; ci < num_cands; ++ci) {
            const Cand& c = cands[ci];
            if (c.pair && !pair_allowed) continue;
            if (c.bn == 64 && is_mx(kind)) continue;                                         // scale blocks span 128 rows
            if (c.pair && is_mxfp8(kind)) continue;                                          // block-scaled fp8 runs on single CTAs
            if (c.bn == 64 && !c.pair && kind == ASCB200_KIND_S8 && !d->trans_b) continue;   // N-contiguous int8 B comes in boxes of 128 columns
            if (c.bn > 64 && n <= c.bn / 2 && (c.pair || c.bn != 128)) continue;             // do not pad N by more than 2x
            const long long n_tiles = (n + c.bn - 1) / c.bn;
            // grouped: the host does not see the counts; a group ends on average half a tile past its last full one
            // (a swapped block costs its share of rows: half a tile on average, like the masked tail it replaces costs in tiles)
            const long long pair_m_tiles = grouped ? (m + 2 * BLOCK_M - 1) / (2 * BLOCK_M) + (groups + 1) / 2 : (m + 2 * BLOCK_M - 1) / (2 * BLOCK_M);
            const long long tiles = c.pair ? pair_m_tiles * n_tiles : m_tiles * n_tiles;
            const long long slots = c.pair ? pair_clusters : sm_count;
            const long long waves = (tiles + slots - 1) / slots;
            double cost = static_cast<double>(waves) * (c.pair ? 2 : 1) * BLOCK_M * c.bn / c.eff / (c.pair ? 2 : 1);
            if (!c.pair && !grouped && !fixed) {  // single-CTA tiles may split K over a cluster (measured speed-ups, see pick_split_k)
                double gain = 1.0;
                pick_split_k(tiles, (k + block_k - 1) / block_k, c.bn, sm_count, &gain);
                cost *= gain;
            }
            if (best < 0 || cost < best) {
                best = cost;
                block_n = c.bn;
                use_pair = c.pair;
            }
        }
    }
    if (const char* force = getenv("ASCB200_PAIR_N")) {
        // testing / tuning override: CTA-pair kernel with this tile width where the kernel supports it
        const int bn = atoi(force);
        if (pair_possible && !is_mx(kind) && (d->trans_b || bn == 256) && bn >= 16 && bn <= 256 && bn % 16 == 0) {
            block_n = bn;
            use_pair = true;
        }
    }
    const long long pair_tiles = (static_cast<long long>((m + 2 * BLOCK_M - 1) / (2 * BLOCK_M)) + (grouped ? groups : 0)) * ((n + block_n - 1) / block_n);

    const int b_box_rows = use_pair ? block_n / 2 : block_n;

    CUtensorMap ta, tb;
    int rc;
    if (!d->trans_a) rc = make_map(&ta, dt, esz, d->a_dev, k / epb, m, 1, lda / epb, static_cast<uint64_t>(lda / epb) * m, row_elems, BLOCK_M);
    else rc = make_map(&ta, dt, esz, d->a_dev, m, k, 1, lda, static_cast<uint64_t>(lda) * k, row_elems, block_k);
    if (rc != ASCB200_OK) return rc;
    const uint64_t g3 = grouped ? groups : 1;
    if (d->trans_b) rc = make_map(&tb, dt, esz, d->b_dev, k / epb, n, g3, ldb / epb, static_cast<uint64_t>(ldb / epb) * n, row_elems, b_box_rows);
    else rc = make_map(&tb, dt, esz, d->b_dev, n, k, g3, ldb, static_cast<uint64_t>(ldb) * k, row_elems, block_k);
    if (rc != ASCB200_OK) return rc;

    GemmParams p = {};
    p.m = m;
    p.n = n;
    p.k = k;
    p.num_k_blocks = (k + block_k - 1) / block_k;
    p.a_mn = d->trans_a ? 1 : 0;
    p.b_mn = d->trans_b ? 0 : 1;
    p.groups = grouped ? groups : 0;
    p.pair_n = block_n;
    p.allow_m64 = !is_mx(kind) && !(getenv("ASCB200_NO_M64") && getenv("ASCB200_NO_M64")[0] == '1');
    // Banded tile order once A alone takes more than half of L2 (measured in the sustained loop: fp16 8192^3, A = 128 MB, 9 %
    // faster; with operands that fit L2 the plain order was 2 to 4 % faster).
    const long long a_bytes = static_cast<long long>(d->m) * d->k * elem_bits(kind) / 8;
    const long long l2_bytes = fixed ? fixed->l2_bytes : st->l2_bytes;
    p.band_m = (!grouped && l2_bytes > 0 && a_bytes > l2_bytes / 2) ? 8 : 0;
    if (const char* band = getenv("ASCB200_BAND_M")) p.band_m = atoi(band);
    p.group_swap = (grouped && use_pair && block_n == 256 && group_swap_ok) ? 1 : 0;
    p.group_counts = reinterpret_cast<const long long*>(group_counts);
    p.status = fixed ? fixed->status_dev : st->status_dev;
    if (linear) {
        e.lin_bias = linear->bias;
        e.lin_bias_f32 = linear->bias_f32;
        e.lin_act = linear->act;
        e.residual = linear->residual;
        e.ld_residual = linear->ld_residual;
        e.order = linear->order;
        e.vec_residual = aligned_to(e.residual, 16) && (e.ld_residual * out_bytes(e.c_dtype)) % 16 == 0;
    }
    p.epi = e;

    if (is_mx(kind)) {
        // Scale factors in the 512-byte chunk order the kernels copy into TMEM (layout documented at retile_scales_kernel):
        // taken as they are when the caller prepacked them (ascb200_mx_scale_prepack: static weights), else re-tiled here
        // into scratch that belongs to `stream`, so that calls on different streams do not overwrite each other's scales.
        const int ks = k / 32;
        const int kc = 2 * ((k + 255) / 256);   // chunks (4 scales each) per 128-row block: the same pitch for every MX kind and for prepacked tensors
        const bool pre_a = (d->scale_flags & ASCB200_SCALE_A_PREPACKED) != 0, pre_b = (d->scale_flags & ASCB200_SCALE_B_PREPACKED) != 0;
        const int rba = (m + 127) / 128, rbb = (n + 127) / 128 + kSfPadBlocks;  // B tiles may read up to two blocks past the last row
        const size_t bytes_a = pre_a ? 0 : static_cast<size_t>(rba) * kc * SF_CHUNK_BYTES, bytes_b = pre_b ? 0 : static_cast<size_t>(rbb) * kc * SF_CHUNK_BYTES;
        uint8_t* scratch = nullptr;
        if (bytes_a + bytes_b > 0) {
            if (fixed) {
                if (bytes_a + bytes_b > fixed->scale_scratch_bytes) return ASCB200_ETOOBIG;
                scratch = fixed->scale_scratch_dev;
            } else {
                void* ptr = nullptr;
                rc = stream_scratch(st, bytes_a + bytes_b, stream, &ptr);
                if (rc != ASCB200_OK) return rc;
                scratch = static_cast<uint8_t*>(ptr);
            }
        }
        const uint8_t* sfa = pre_a ? static_cast<const uint8_t*>(d->scale_a_dev) : scratch;
        const uint8_t* sfb = pre_b ? static_cast<const uint8_t*>(d->scale_b_dev) : scratch + bytes_a;
        if (!aligned_to(sfa, 16) || !aligned_to(sfb, 16)) return ASCB200_EALIGN;
        if (scratch) {
            const int kc_tiles = (kc + 7) / 8;
            const int blocks_a = pre_a ? 0 : rba * kc_tiles, blocks_b = pre_b ? 0 : rbb * kc_tiles;
            ASCB200_CUDA(launch_pdl(retile_scales_kernel, dim3(blocks_a + blocks_b), dim3(256), 0, stream, static_cast<const uint8_t*>(d->scale_a_dev),
                                    reinterpret_cast<uint32_t*>(scratch), m, pre_a ? 0 : rba, static_cast<const uint8_t*>(d->scale_b_dev),
                                    reinterpret_cast<uint32_t*>(scratch + bytes_a), n, ks, kc, kc_tiles,
                                    ((d->scale_flags & ASCB200_SCALE_A_PAIRED) ? 1 : 0) | ((d->scale_flags & ASCB200_SCALE_B_PAIRED) ? 2 : 0)));
        }
        p.sfa = sfa;
        p.sfb = sfb;
        p.sf_kc = kc;
    }

    const long long max_tiles = grouped ? (static_cast<long long>((m + BLOCK_M - 1) / BLOCK_M) + groups) * ((n + block_n - 1) / block_n)
                                        : static_cast<long long>((m + BLOCK_M - 1) / BLOCK_M) * ((n + block_n - 1) / block_n);
    const int grid = static_cast<int>(std::min<long long>(max_tiles, sm_count));
    // Few tiles and a long K: clusters of 2 or 4 CTAs share each tile and split its K blocks (a K block cannot take less than
    // about 370 cycles whatever the tile's width, so a small problem's time is its number of K blocks); the leader adds the
    // others' accumulators in rank order.  Never for grouped calls or calls that bring their own device resources.
    if (!use_pair && !grouped && !fixed) {
        int sk = pick_split_k(max_tiles, p.num_k_blocks, block_n, sm_count);
        if (const char* force = getenv("ASCB200_SPLIT_K")) {
            const int v = atoi(force);
            sk = (v == 2 || v == 4 || v == 8) && max_tiles * v <= sm_count ? v : 0;
        }
        p.split_k = sk;
    }

    const uint32_t a_mn = p.a_mn, b_mn = p.b_mn;
    if (use_pair) {
        const int clusters = static_cast<int>(std::min<long long>(pair_tiles, pair_clusters));
        if (kind == ASCB200_KIND_MXFP4) {
            // the re-tiled scales as rank-2 tensors [chunk][128 x u32] for tile loads
            CUtensorMap tsfa, tsfb;
            rc = make_sf_map(&tsfa, p.sfa, static_cast<uint64_t>((m + 127) / 128) * p.sf_kc, 2);
            if (rc == ASCB200_OK) rc = make_sf_map(&tsfb, p.sfb, static_cast<uint64_t>((n + 127) / 128 + kSfPadBlocks) * p.sf_kc, 2);
            if (rc != ASCB200_OK) return rc;
            p.idesc = make_idesc_mxf4(2 * BLOCK_M, 192);
            return launch_gemm_pair<KIND_MXF4, 192>(ta, tb, tsfa, tsfb, outs, p, clusters, stream);
        }
        if (kind == ASCB200_KIND_S8) {
            p.idesc = make_idesc(2, 1, 1, a_mn, b_mn, 2 * BLOCK_M, block_n);
            if (linear) return launch_linear_gemm(KIND_I8, true, block_n, ta, tb, outs, p, clusters, stream);
            CUtensorMap tx32 = ta;
            if (p.group_swap) {
                // the weights as the 256-row operand, rows of A as the narrow one (its N field is filled in per block);
                // A once more with boxes of 32 rows, for blocks that hold fewer than 97 rows per CTA
                p.idesc_swap = make_idesc(2, 1, 1, b_mn, a_mn, 2 * BLOCK_M, 0);
                rc = make_map(&tx32, dt, esz, d->a_dev, k, m, 1, lda, static_cast<uint64_t>(lda) * m, row_elems, 32);
                if (rc != ASCB200_OK) return rc;
            }
            return launch_gemm_pair<KIND_I8, 256>(ta, tb, tx32, tb, outs, p, clusters, stream);
        }
        const uint32_t fmt = kind == ASCB200_KIND_BF16 ? 1u : 0u;
        p.idesc = make_idesc(1, fmt, fmt, a_mn, b_mn, 2 * BLOCK_M, block_n);
        if (linear) return launch_linear_gemm(KIND_F16, true, block_n, ta, tb, outs, p, clusters, stream);
        return launch_gemm_pair<KIND_F16, 256>(ta, tb, ta, tb, outs, p, clusters, stream);
    }
    if (is_mxfp8(kind)) {
        const uint32_t fmt = kind == ASCB200_KIND_MXFP8_E5M2 ? 1u : 0u;
        p.idesc = make_idesc_mxf8(fmt, fmt, a_mn, b_mn, BLOCK_M, block_n);
        if (block_n == 256) return launch_gemm<KIND_MXF8, 256>(ta, tb, outs, p, grid, stream);
        if (block_n == 192) return launch_gemm<KIND_MXF8, 192>(ta, tb, outs, p, grid, stream);
        return launch_gemm<KIND_MXF8, 128>(ta, tb, outs, p, grid, stream);
    }
    switch (kind) {
        case ASCB200_KIND_F16:
        case ASCB200_KIND_BF16: {
            const uint32_t fmt = kind == ASCB200_KIND_BF16 ? 1u : 0u;
            p.idesc = make_idesc(1, fmt, fmt, a_mn, b_mn, BLOCK_M, block_n);
            if (linear) return launch_linear_gemm(KIND_F16, false, block_n, ta, tb, outs, p, grid, stream);
            if (block_n == 256) return launch_gemm<KIND_F16, 256>(ta, tb, outs, p, grid, stream);
            if (block_n == 128) return launch_gemm<KIND_F16, 128>(ta, tb, outs, p, grid, stream);
            return launch_gemm<KIND_F16, 64>(ta, tb, outs, p, grid, stream);
        }
        case ASCB200_KIND_S8:
            p.idesc = make_idesc(2, 1, 1, a_mn, b_mn, BLOCK_M, block_n);
            if (linear) return launch_linear_gemm(KIND_I8, false, block_n, ta, tb, outs, p, grid, stream);
            if (block_n == 256) return launch_gemm<KIND_I8, 256>(ta, tb, outs, p, grid, stream);
            if (block_n == 128) return launch_gemm<KIND_I8, 128>(ta, tb, outs, p, grid, stream);
            return launch_gemm<KIND_I8, 64>(ta, tb, outs, p, grid, stream);
        default:
            p.idesc = make_idesc_mxf4(BLOCK_M, block_n);
            if (block_n == 256) return launch_gemm<KIND_MXF4, 256>(ta, tb, outs, p, grid, stream);
            if (block_n == 192) return launch_gemm<KIND_MXF4, 192>(ta, tb, outs, p, grid, stream);
            return launch_gemm<KIND_MXF4, 128>(ta, tb, outs, p, grid, stream);
    }
}

namespace {

// ---- allocation-free MXFP4 variant ------------------------------------------------------------------
// Scratch of ascb200_gemm_mxfp4_noalloc: 256 bytes for the status word of the bounded waits, then the
// re-tiled scale factors.  The array lives in the library image: every GPU that loads the library
// holds these bytes until the process exits.
constexpr size_t NOALLOC_HEAD_BYTES = 256;
constexpr size_t NOALLOC_SCALE_BYTES = ASCB200_NOALLOC_MAX_SCALE_BYTES;
static __device__ __align__(256) uint8_t g_noalloc_scratch[NOALLOC_HEAD_BYTES + NOALLOC_SCALE_BYTES];

struct NoAllocDevice {
    bool ready = false;
    uint8_t* base = nullptr;  // device address of g_noalloc_scratch on this device
    int sm_count = 0;
};
NoAllocDevice g_noalloc_dev[16];
std::mutex g_noalloc_mu;

// Once per device, with that device current: resolve the device address of the array.  In host code
// the symbol itself is only a stand-in and must never be handed to a kernel.
int noalloc_setup(NoAllocDevice** out)
{
    int dev = -1;
    ASCB200_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 16) return ASCB200_EINVAL;
    std::lock_guard<std::mutex> lock(g_noalloc_mu);
    NoAllocDevice* nd = &g_noalloc_dev[dev];
    if (!nd->ready) {
        int major = 0, sms = 0;
        ASCB200_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
        if (major != 10) return ASCB200_ENODEV;
        ASCB200_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        void* ptr = nullptr;
        ASCB200_CUDA(cudaGetSymbolAddress(&ptr, g_noalloc_scratch));
        if (!ptr) return ASCB200_ECUDA;
        nd->base = static_cast<uint8_t*>(ptr);
        nd->sm_count = sms;
        nd->ready = true;
    }
    *out = nd;
    return ASCB200_OK;
}

int run_gemm_mxfp4_noalloc(const ascb200_gemm_desc* d, cudaStream_t stream)
{
    if (!d) return ASCB200_EINVAL;
    if (d->kind != ASCB200_KIND_MXFP4) return ASCB200_EUNSUPPORTED;
    NoAllocDevice* nd = nullptr;
    int rc = noalloc_setup(&nd);
    if (rc != ASCB200_OK) return rc;
    FixedResources fixed;
    fixed.status_dev = reinterpret_cast<uint32_t*>(nd->base);
    fixed.scale_scratch_dev = nd->base + NOALLOC_HEAD_BYTES;
    fixed.scale_scratch_bytes = NOALLOC_SCALE_BYTES;
    fixed.sm_count = nd->sm_count;
    fixed.l2_bytes = 0;
    // The array keeps whatever the previous call left.  Nothing in it has to start at zero: the re-tiling kernel rewrites
    // every scale byte the GEMM reads, and the status word is a latch (zero when the library image is loaded, set by an
    // expired wait, read and cleared by ascb200_noalloc_status).
    return run_gemm(d, nullptr, 0, stream, &fixed);
}

int noalloc_status(cudaStream_t stream, uint32_t* status_host)
{
    NoAllocDevice* nd = nullptr;
    int rc = noalloc_setup(&nd);
    if (rc != ASCB200_OK) return rc;
    uint32_t v = 0;
    ASCB200_CUDA(cudaMemcpyAsync(&v, nd->base, sizeof(v), cudaMemcpyDeviceToHost, stream));
    ASCB200_CUDA(cudaStreamSynchronize(stream));
    if (status_host) *status_host = v;
    if (v != 0) {
        ASCB200_CUDA(cudaMemsetAsync(nd->base, 0, sizeof(v), stream));
        return ASCB200_ETIMEOUT;
    }
    return ASCB200_OK;
}

// Re-tiles one scale tensor [rows, k / 32] into the chunk order of the kernels, padding blocks included.
int mx_scale_prepack(const void* scale_dev, int rows, int k, int paired, void* out_dev, size_t out_bytes, cudaStream_t stream)
{
    if (!scale_dev || !out_dev || rows <= 0 || k <= 0 || k % 64 != 0) return ASCB200_EINVAL;
    if (!aligned_to(out_dev, 16)) return ASCB200_EALIGN;
    const int block_k = 256;
    const int kc = 2 * ((k + block_k - 1) / block_k);
    const int rb = (rows + 127) / 128 + kSfPadBlocks;
    if (out_bytes < static_cast<size_t>(rb) * kc * SF_CHUNK_BYTES) return ASCB200_EINVAL;
    const int kc_tiles = (kc + 7) / 8;
    ASCB200_CUDA(launch_pdl(retile_scales_kernel, dim3(rb * kc_tiles), dim3(256), 0, stream, static_cast<const uint8_t*>(scale_dev),
                            static_cast<uint32_t*>(out_dev), rows, rb, static_cast<const uint8_t*>(nullptr), static_cast<uint32_t*>(nullptr), 0, k / 32,
                            kc, kc_tiles, paired ? 1 : 0));
    return ASCB200_OK;
}

}  // namespace
}  // namespace gemm
}  // namespace ascb200

extern "C" {

int ascb200_noalloc_status(void* stream, uint32_t* status_host) { return ascb200::gemm::noalloc_status(static_cast<cudaStream_t>(stream), status_host); }

size_t ascb200_mx_scale_prepacked_bytes(int32_t rows, int32_t k)
{
    if (rows <= 0 || k <= 0) return 0;
    return static_cast<size_t>((rows + 127) / 128 + ascb200::gemm::kSfPadBlocks) * (2 * ((k + 255) / 256)) * ascb200::gemm::SF_CHUNK_BYTES;
}

int ascb200_mx_scale_prepack(const void* scale_dev, int32_t rows, int32_t k, int32_t paired, void* out_dev, size_t out_bytes, void* stream)
{
    if (!ascb200::current_state()) return ASCB200_ENODEV;
    return ascb200::gemm::mx_scale_prepack(scale_dev, rows, k, paired, out_dev, out_bytes, static_cast<cudaStream_t>(stream));
}

int ascb200_gemm_mxfp4_noalloc(const ascb200_gemm_desc* desc, void* stream)
{
    return ascb200::gemm::run_gemm_mxfp4_noalloc(desc, static_cast<cudaStream_t>(stream));
}

int ascb200_gemm(const ascb200_gemm_desc* desc, void* stream)
{
    return ascb200::gemm::run_gemm(desc, nullptr, 0, static_cast<cudaStream_t>(stream));
}

int ascb200_grouped_gemm(const ascb200_gemm_desc* desc, const int64_t* group_counts_dev, int32_t groups, void* stream)
{
    if (groups <= 0) return groups == 0 ? ASCB200_OK : ASCB200_EINVAL;
    return ascb200::gemm::run_gemm(desc, group_counts_dev, groups, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

