// Gradient of an activation (gated or not) quantised for both products of a backward pass, and the
// transposing MX quantiser.
//
// D = dh up f'(gate) | dh f(gate)   (gated), or dh f'(gate)
// is needed twice as an MX operand: with blocks of 32 along its rows (dX = D Wt^T sums over the
// features) and along its columns (dW = D^T X sums over the rows of D). Both come from one pass
// over dh, gate and up, which HBM bounds: a CTA takes 128 rows x 64 columns, computes D in f32
// once, quantises and stores the row blocks from registers, leaves D in shared memory and reads it
// back by columns for the transposed operand. Loads are 128-byte row segments, all of a tile
// issued before the first use; 8 lanes hold a row segment, so a row block of 32 is four lanes. In
// the second step a thread holds one column's 32 rows, i.e. one whole block, and stores its 32
// codes as two 16-byte vectors.
#include "common.cuh"
#include "data_types.cuh"
#include "mx_block.cuh"
#include "reduce.cuh"

namespace {

namespace dt = ptxstd::data_types;
namespace mx = ptxstd::mx;

constexpr uint32_t kRows = 128, kCols = 64, kThreads = 256;
constexpr uint32_t kPasses = kRows / 32;  // 8 warps x 4 rows a pass
enum Mode { kTranspose = 0, kPlain = 1, kGated = 2 };

struct Params {
    const uint16_t *dh, *gate, *up;  // kTranspose: gate is x
    uint8_t *q, *sf, *qt, *sft;
    float* partial;  // [row tiles][W] column sums, or null
    uint32_t rows, cols, W, R;  // W columns of D, R = rows rounded up to 32
    uint32_t col_tiles, act, type;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        o[2 * k] = dt::bf16_lo(w[k]);
        o[2 * k + 1] = dt::bf16_hi(w[k]);
    }
}

// Eight values of a row to the tile in shared memory. The halves are swapped for lanes 4..7 of a
// row so that eight lanes' 16-byte stores fall into different banks.
__device__ __forceinline__ void put8(float* row, uint32_t l, const float (&v)[8]) {
    float4* p = reinterpret_cast<float4*>(row + 8 * l);
    const float4 lo = make_float4(v[0], v[1], v[2], v[3]);
    const float4 hi = make_float4(v[4], v[5], v[6], v[7]);
    const uint32_t h = (l >> 2) & 1u;
    p[h] = h ? hi : lo;
    p[h ^ 1u] = h ? lo : hi;
}

// One row block (four lanes) of D at (row, first column col of this lane's eight values).
__device__ __forceinline__ void row_block(const Params& p, const float (&v)[8], uint32_t row,
                                          uint32_t col, bool on, bool in_tiles, uint32_t lane) {
    const mx::Scale sc = mx::scale_of(mx::amax_quad(mx::amax_of(v)), mx::emax_of(p.type));
    if (on)
        *reinterpret_cast<uint2*>(p.q + static_cast<size_t>(row) * p.W + col) =
            mx::pack8(p.type, v, sc.inv);
    if ((lane & 3u) == 0 && in_tiles) {
        const uint32_t s = col / 32;
        p.sf[mx::word_offset(row, s >> 2, mx::tiles_k(p.W / 32)) + (s & 3u)] =
            on ? static_cast<uint8_t>(sc.code) : 0;
    }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads)
    act_backward_kernel(const __grid_constant__ Params p) {
    constexpr int kTiles = MODE == kGated ? 2 : 1;
    extern __shared__ float4 smem_raw[];
    float* const tile = reinterpret_cast<float*>(smem_raw);  // [kTiles][kRows][kCols]
    __shared__ float sums[4][kCols];
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t ct = blockIdx.x % p.col_tiles, rt = blockIdx.x / p.col_tiles;
    const uint32_t row0 = rt * kRows, col0 = ct * kCols;
    const uint32_t l = lane & 7u, col = col0 + 8 * l;

    ptxstd::pdl_launch_dependents();
    ptxstd::pdl_wait();

    {
        uint4 gv[kPasses], dv[kPasses], uv[kPasses];
#pragma unroll
        for (uint32_t i = 0; i < kPasses; ++i) {
            const uint32_t row = row0 + i * 32 + warp * 4 + (lane >> 3);
            gv[i] = dv[i] = uv[i] = make_uint4(0, 0, 0, 0);
            if (row < p.rows && col < p.cols) {
                const size_t at = static_cast<size_t>(row) * p.cols + col;
                gv[i] = *reinterpret_cast<const uint4*>(p.gate + at);
                if (MODE != kTranspose) dv[i] = *reinterpret_cast<const uint4*>(p.dh + at);
                if (MODE == kGated) uv[i] = *reinterpret_cast<const uint4*>(p.up + at);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kPasses; ++i) {
            const uint32_t r = i * 32 + warp * 4 + (lane >> 3), row = row0 + r;
            float g[8], d[8];
            unpack8(gv[i], g);
            if constexpr (MODE == kTranspose) {
                put8(tile + r * kCols, l, g);
            } else {
                const bool on = row < p.rows && col < p.cols, in_tiles = col < p.cols;
                float a[8], b[8];
                unpack8(dv[i], d);
                switch (p.act) {
#define PTXSTD_CASE(K)                                                              \
    case K:                                                                         \
        _Pragma("unroll") for (int k = 0; k < 8; ++k) mx::act_grad(K, g[k], a[k], b[k]); \
        break;
                    PTXSTD_CASE(PTXSTD_ACT_RELU)
                    PTXSTD_CASE(PTXSTD_ACT_SILU)
                    PTXSTD_CASE(PTXSTD_ACT_GELU)
                    PTXSTD_CASE(PTXSTD_ACT_GELU_TANH)
#undef PTXSTD_CASE
                default:
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        a[k] = g[k];
                        b[k] = 1.0f;
                    }
                }
                if constexpr (MODE == kGated) {
                    float u[8];
                    unpack8(uv[i], u);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        b[k] *= d[k] * u[k];  // dgate
                        a[k] *= d[k];         // dup
                    }
                    put8(tile + r * kCols, l, b);
                    put8(tile + (kRows + r) * kCols, l, a);
                    row_block(p, b, row, col, on, in_tiles, lane);
                    row_block(p, a, row, p.cols + col, on, in_tiles, lane);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) b[k] *= d[k];
                    put8(tile + r * kCols, l, b);
                    row_block(p, b, row, col, on, in_tiles, lane);
                }
            }
        }
    }
    __syncthreads();

    // transposed: thread = (column f, row block b)
    const uint32_t f = tid & (kCols - 1), b = tid / kCols;
    const uint32_t t0 = row0 + 32 * b;
    const size_t kt = mx::tiles_k(p.R / 32);
    const uint32_t emax = mx::emax_of(p.type);
#pragma unroll
    for (int h = 0; h < kTiles; ++h) {
        const float* src = tile + (h * kRows + 32 * b) * kCols + f;
        float v[32];
        float sum = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) {
            v[i] = src[i * kCols];
            sum += v[i];
        }
        const mx::Scale sc = mx::scale_of(mx::amax_of(v), emax);
        const uint32_t feature = h * p.cols + col0 + f;
        if (col0 + f < p.cols) {
            if (t0 < p.R) {
                uint4* dst = reinterpret_cast<uint4*>(p.qt + static_cast<size_t>(feature) * p.R + t0);
#pragma unroll
                for (uint32_t c = 0; c < 2; ++c) {
                    const uint2 lo = mx::pack8(p.type, v + 16 * c, sc.inv);
                    const uint2 hi = mx::pack8(p.type, v + 16 * c + 8, sc.inv);
                    dst[c] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
            }
            p.sft[mx::word_offset(feature, rt, kt) + b] =
                t0 < p.R ? static_cast<uint8_t>(sc.code) : 0;
        }
        if (MODE != kTranspose && p.partial) {
            sums[b][f] = sum;
            __syncthreads();
            if (b == 0 && col0 + f < p.cols)
                p.partial[static_cast<size_t>(rt) * p.W + feature] =
                    (sums[0][f] + sums[1][f]) + (sums[2][f] + sums[3][f]);
            if (h + 1 < kTiles) __syncthreads();
        }
    }

    // padding of the scale tiles: the CTAs of the first column tile write it
    if (ct == 0) {
        const uint32_t w_rows = static_cast<uint32_t>(mx::padded_rows(p.W));
        for (uint32_t r = p.W + tid; r < w_rows; r += kThreads)
            *reinterpret_cast<uint32_t*>(p.sft + mx::word_offset(r, rt, kt)) = 0;
        if (MODE != kTranspose) {
            const uint32_t blocks = p.W / 32;
            const size_t k_tiles = mx::tiles_k(blocks);
            if (tid < kRows && (blocks & 3u))
                for (uint32_t s = blocks & 3u; s < 4; ++s)
                    p.sf[mx::word_offset(row0 + tid, k_tiles - 1, k_tiles) + s] = 0;
        }
    }
}

template <int MODE>
int launch(Params& p, cudaStream_t stream) {
    p.R = (p.rows + 31) / 32 * 32;
    p.col_tiles = (p.cols + kCols - 1) / kCols;
    const uint64_t tiles =
        static_cast<uint64_t>(p.col_tiles) * ((static_cast<uint64_t>(p.rows) + kRows - 1) / kRows);
    if (tiles >= (1ull << 31)) return PTXSTD_EINVAL;
    constexpr int kSmem = (MODE == kGated ? 2 : 1) * kRows * kCols * 4;
    const int st = ptxstd::set_max_dynamic_smem(
        reinterpret_cast<const void*>(act_backward_kernel<MODE>), kSmem);
    if (st) return st;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    ptxstd::set_pdl(cfg, attr, static_cast<uint32_t>(tiles), kThreads, stream);
    cfg.dynamicSmemBytes = kSmem;
    if (cudaLaunchKernelEx(&cfg, act_backward_kernel<MODE>, p) != cudaSuccess) return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

bool bad(const void* p) { return !p || !ptxstd::aligned16(p); }

bool sizes_ok(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 && rows < (1ll << 31) - 128 && cols < (1ll << 30);
}

}  // namespace

extern "C" size_t ptxstd_act_backward_mx_workspace_bytes(int64_t rows, int64_t cols, int gated,
                                                         int with_dbias) {
    if (!with_dbias || !sizes_ok(rows, cols)) return 0;
    return static_cast<size_t>((rows + kRows - 1) / kRows) * static_cast<size_t>(cols) *
           (gated ? 2 : 1) * 4;
}

extern "C" int ptxstd_act_backward_mx(int act, const uint16_t* d_dh, const uint16_t* d_gate,
                                      const uint16_t* d_up, int64_t rows, int64_t cols,
                                      int elem_type, uint8_t* d_q, uint8_t* d_sf, uint8_t* d_qt,
                                      uint8_t* d_sft, float* d_dbias, void* d_workspace,
                                      size_t workspace_bytes, ptxstd_stream stream) {
    if (!sizes_ok(rows, cols) || cols % 32) return PTXSTD_EINVAL;
    if (act < PTXSTD_ACT_NONE || act > PTXSTD_ACT_GELU_TANH) return PTXSTD_EINVAL;
    if (elem_type != PTXSTD_MX_E4M3 && elem_type != PTXSTD_MX_E5M2) return PTXSTD_EINVAL;
    if (bad(d_dh) || bad(d_gate) || bad(d_q) || bad(d_sf) || bad(d_qt) || bad(d_sft) ||
        !ptxstd::aligned16(d_up) || !ptxstd::aligned16(d_dbias))
        return PTXSTD_EINVAL;
    Params p = {};
    p.dh = d_dh;
    p.gate = d_gate;
    p.up = d_up;
    p.q = d_q;
    p.sf = d_sf;
    p.qt = d_qt;
    p.sft = d_sft;
    p.rows = static_cast<uint32_t>(rows);
    p.cols = static_cast<uint32_t>(cols);
    p.W = p.cols * (d_up ? 2u : 1u);
    p.act = static_cast<uint32_t>(act);
    p.type = static_cast<uint32_t>(elem_type);
    if (d_dbias) {
        if (bad(d_workspace) || workspace_bytes < ptxstd_act_backward_mx_workspace_bytes(
                                                      rows, cols, d_up != nullptr, 1))
            return PTXSTD_EINVAL;
        p.partial = static_cast<float*>(d_workspace);
    }
    auto s = static_cast<cudaStream_t>(stream);
    const int st = d_up ? launch<kGated>(p, s) : launch<kPlain>(p, s);
    if (st || !d_dbias) return st;
    ptxstd::Reduce r = {};
    r.partial = p.partial;
    r.P = (p.rows + kRows - 1) / kRows;
    r.sums = 1;
    r.cols = p.W;
    r.o0 = d_dbias;
    return ptxstd::launch_reduce(r, s);
}

extern "C" int ptxstd_quantize_mx_t(const uint16_t* d_x, int64_t rows, int64_t cols, int elem_type,
                                    uint8_t* d_qt, uint8_t* d_sft, ptxstd_stream stream) {
    if (!sizes_ok(rows, cols) || cols % 8) return PTXSTD_EINVAL;
    if (elem_type != PTXSTD_MX_E4M3 && elem_type != PTXSTD_MX_E5M2) return PTXSTD_EINVAL;
    if (bad(d_x) || bad(d_qt) || bad(d_sft)) return PTXSTD_EINVAL;
    Params p = {};
    p.gate = d_x;
    p.qt = d_qt;
    p.sft = d_sft;
    p.rows = static_cast<uint32_t>(rows);
    p.cols = p.W = static_cast<uint32_t>(cols);
    p.type = static_cast<uint32_t>(elem_type);
    return launch<kTranspose>(p, static_cast<cudaStream_t>(stream));
}
