// Gradient of an activation (gated or not) quantised for both products of a backward pass, and the
// transposing MX quantiser.
//
// D = dh up f'(gate) | dh f(gate)   (gated), or dh f'(gate)
// is needed twice as an MX operand: with blocks of 32 along its rows (dX = D Wt^T sums over the
// features) and along its columns (dW = D^T X sums over the rows of D). Both come from one pass
// over dh, gate and up, which HBM bounds: a CTA takes 64 rows x 64 columns, computes D in f32
// once, quantises and stores the row blocks from registers, leaves D in shared memory and reads it
// back by columns for the transposed operand. Loads are 128-byte row segments, all of a tile
// issued before the first use; 8 lanes hold a row segment, so a row block of 32 is four lanes. In
// the second step a thread holds one column's 32 rows, i.e. one whole block, and stores its 32
// codes in one instruction; the column's other 32 rows belong to the neighbouring lane, so that a
// pair writes 64 adjacent bytes, its two scales as one half-word, and adds its sums by a shuffle.
// (As two 16-byte stores, with a column's halves in different warps, the requests to L2 bound the
// kernel: ReLU 82 us instead of 71 us, the transposing quantiser of 8192 x 8192 50 us instead of
// 41 us, gated 99 us instead of 88 us.)
// 4096 x 16384, E5M2, column sums included, results of successive calls in different buffers, under
// load: 407 MB in 71 us with ReLU (0.88 of the measured copy rate), 89 us with GELU, which takes 31
// instructions per element to ReLU's 21 and so the issue slots to three quarters (ncu); at the
// clock of an idle GPU 67 and 80 us. Gated, SiLU, 4096 x 10240: 425 MB in 88 us (0.74). The
// transposing quantiser of 8192 x 8192: 204 MB in 41 us (0.76). Without effect or slower: other
// orders of the tiles, prefetching a later tile to L2, a persistent form that copies the next tile
// to shared memory meanwhile (gated 81 us instead of 84 us, GELU 106 instead of 83).
#include "common.cuh"
#include "data_types.cuh"
#include "mx_block.cuh"
#include "reduce.cuh"

namespace {

namespace dt = ptxstd::data_types;
namespace mx = ptxstd::mx;

constexpr uint32_t kRows = 64, kCols = 64, kThreads = 128;
constexpr uint32_t kPassRows = kThreads / 8;  // eight lanes to a row's 64 columns
constexpr uint32_t kPasses = kRows / kPassRows;
enum Mode { kTranspose = 0, kPlain = 1, kGated = 2 };

struct Params {
    const uint16_t *dh, *gate, *up;  // kTranspose: gate is x
    uint8_t *q, *sf, *qt, *sft;
    float* partial;  // [row tiles][W] column sums, or null
    uint32_t rows, cols, W, R;  // W columns of D, R = rows rounded up to 32
    uint32_t col_tiles, act, type;
    bool wide;  // qt is 32-byte aligned
};

using ptxstd::f32x2;
using ptxstd::mul2;
using ptxstd::Oct;
using ptxstd::widen;

// The tile in shared memory, [row][64] f32 as 16 slots of four columns. Slot s of a row in block b
// of 32 rows sits at s ^ (s / 8) ^ 4 b: then the eight lanes of a quarter-warp, which hold slots 0,
// 2, .. 14 (then 1, 3, .. 15) of one row, store into different banks. A column keeps its place in
// every row of a block, and a warp that reads 16 neighbouring columns in both blocks finds one
// block's in the other half of the banks, so reading is free of conflicts too.
__device__ __forceinline__ uint32_t slot_of(uint32_t s, uint32_t b) { return s ^ (s >> 3) ^ (4 * b); }

// Eight values (lane l of a row's eight) to the tile; b: the row's block of 32.
__device__ __forceinline__ void put8(float4* row, uint32_t l, uint32_t b, const float (&v)[8]) {
    row[slot_of(2 * l, b)] = make_float4(v[0], v[1], v[2], v[3]);
    row[slot_of(2 * l + 1, b)] = make_float4(v[4], v[5], v[6], v[7]);
}

// 32 codes of one column.
__device__ __forceinline__ void store32(uint8_t* dst, const uint2 (&c)[4], bool wide) {
    if (wide)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst),
                     "r"(c[0].x), "r"(c[0].y), "r"(c[1].x), "r"(c[1].y), "r"(c[2].x), "r"(c[2].y),
                     "r"(c[3].x), "r"(c[3].y)
                     : "memory");
    else {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(c[0].x, c[0].y, c[1].x, c[1].y);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(c[2].x, c[2].y, c[3].x, c[3].y);
    }
}

// One row block (four lanes) of D: eight codes to q, the block's scale to sf (first lane).
__device__ __forceinline__ void row_block(uint32_t type, const float (&v)[8], bool on, uint8_t* q,
                                          bool first, uint8_t* sf) {
    const mx::Scale sc = mx::scale_of(mx::amax_quad(mx::amax_of(v)), mx::emax_of(type));
    if (on) *reinterpret_cast<uint2*>(q) = mx::pack8(type, v, sc.inv);
    if (first) *sf = on ? static_cast<uint8_t>(sc.code) : 0;
}

// Blocks per SM asked of the compiler: enough registers that all of a tile's loads are in flight at
// once. Gated, SiLU, 4096 x 10240: 84 us with 5 (96 registers), 110 us with 6 (80 registers, loads
// in turn with their use). Ungated, GELU, 4096 x 16384: 81 us with 9, 83 us with 8, 88 us with 10.
template <int MODE>
__global__ void __launch_bounds__(kThreads, MODE == kGated ? 5 : 9)
    act_backward_kernel(const __grid_constant__ Params p) {
    constexpr int kTiles = MODE == kGated ? 2 : 1;
    extern __shared__ float4 smem_raw[];
    float4* const tile = smem_raw;  // [kTiles][kRows][kCols / 4]
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t ct = blockIdx.x % p.col_tiles, rt = blockIdx.x / p.col_tiles;
    const uint32_t row0 = rt * kRows, col0 = ct * kCols;
    const uint32_t l = lane & 7u, col = col0 + 8 * l;

    ptxstd::pdl_launch_dependents();
    ptxstd::pdl_wait();

    {
        // pass i: rows r, r + kPassRows, ... of the tile
        const uint32_t r = warp * 4 + (lane >> 3), row = row0 + r;
        const bool col_on = col < p.cols;
        const size_t at = static_cast<size_t>(row) * p.cols + col, step = static_cast<size_t>(kPassRows) * p.cols;
        uint4 gv[kPasses], dv[kPasses], uv[kPasses];
        auto load = [&](uint32_t i) {
            gv[i] = *reinterpret_cast<const uint4*>(p.gate + at + i * step);
            if (MODE != kTranspose) dv[i] = *reinterpret_cast<const uint4*>(p.dh + at + i * step);
            if (MODE == kGated) uv[i] = *reinterpret_cast<const uint4*>(p.up + at + i * step);
        };
        if (row0 + kRows <= p.rows && col0 + kCols <= p.cols) {
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) load(i);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) {
                gv[i] = dv[i] = uv[i] = make_uint4(0, 0, 0, 0);
                if (row + kPassRows * i < p.rows && col_on) load(i);
            }
        }
        float4* const dst = tile + r * (kCols / 4);
        if constexpr (MODE == kTranspose) {
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) {
                float v[8];
                ptxstd::flatten(widen(gv[i]), v);
                put8(dst + i * kPassRows * (kCols / 4), l, i * kPassRows / 32, v);
            }
        } else {
            const size_t k_tiles = mx::tiles_k(p.W / 32);
            uint8_t* const q = p.q + static_cast<size_t>(row) * p.W + col;
            const uint32_t s0 = col / 32, s1 = (p.cols + col) / 32;
            const bool first = (lane & 3u) == 0 && col_on;
            // the tile's rows lie in one 128-row scale tile
            uint8_t* const sf = p.sf + (row0 >> 7) * k_tiles * 512;
            uint8_t* const sf0 = sf + (s0 >> 2) * 512 + (s0 & 3u);
            uint8_t* const sf1 = sf + (s1 >> 2) * 512 + (s1 & 3u);
            const uint32_t rr = row & 127u;
            mx::with_act(p.act, [&](auto kind) {
#pragma unroll
                for (uint32_t i = 0; i < kPasses; ++i) {
                    const uint32_t ri = rr + kPassRows * i, at_sf = (ri & 31u) * 16 + (ri >> 5) * 4;
                    const bool on = row + kPassRows * i < p.rows && col_on;
                    const Oct g = widen(gv[i]), d = widen(dv[i]);
                    Oct a, b;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        mx::act_grad2<decltype(kind)::value>(g.v[k], a.v[k], b.v[k]);
                        b.v[k] = mul2(b.v[k], d.v[k]);
                    }
                    if constexpr (MODE == kGated) {
                        const Oct u = widen(uv[i]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            b.v[k] = mul2(b.v[k], u.v[k]);  // dgate
                            a.v[k] = mul2(a.v[k], d.v[k]);  // dup
                        }
                    }
                    float v[8];
                    ptxstd::flatten(b, v);
                    put8(dst + i * kPassRows * (kCols / 4), l, i * kPassRows / 32, v);
                    row_block(p.type, v, on, q + i * static_cast<size_t>(kPassRows) * p.W, first,
                              sf0 + at_sf);
                    if constexpr (MODE == kGated) {
                        ptxstd::flatten(a, v);
                        put8(dst + (kRows + i * kPassRows) * (kCols / 4), l, i * kPassRows / 32, v);
                        row_block(p.type, v, on, q + i * static_cast<size_t>(kPassRows) * p.W + p.cols,
                                  first, sf1 + at_sf);
                    }
                }
            });
        }
    }
    __syncthreads();

    // transposed: thread = (column f, row block b), the two blocks of a column in neighbouring lanes
    const uint32_t f = tid >> 1, b = tid & 1u;
    const uint32_t t0 = row0 + 32 * b;
    const size_t kt = mx::tiles_k(p.R / 32);
    const uint32_t emax = mx::emax_of(p.type);
    const float* const column =
        reinterpret_cast<const float*>(tile) + 4 * slot_of(f >> 2, b) + (f & 3u);
    const bool f_on = col0 + f < p.cols;
#pragma unroll
    for (int h = 0; h < kTiles; ++h) {
        const float* src = column + (h * kRows + 32 * b) * kCols;
        float v[32];
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) v[i] = src[i * kCols];
        const mx::Scale sc = mx::scale_of(mx::amax_of(v), emax);
        const uint32_t feature = h * p.cols + col0 + f;
        if (f_on && t0 < p.R) {
            uint2 c[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) c[k] = mx::pack8(p.type, v + 8 * k, sc.inv);
            store32(p.qt + static_cast<size_t>(feature) * p.R + t0, c, p.wide);
        }
        const uint32_t code = t0 < p.R ? sc.code : 0;
        const uint32_t other = __shfl_down_sync(0xffffffffu, code, 1);
        if (f_on && b == 0)
            *reinterpret_cast<uint16_t*>(p.sft + mx::word_offset(feature, t0 >> 7, kt) +
                                         ((t0 >> 5) & 3u)) = static_cast<uint16_t>(code | other << 8);
        if (MODE != kTranspose && p.partial) {
            f32x2 sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < 32; i += 2)
                sum = ptxstd::add2(sum, ptxstd::pack2f(v[i], v[i + 1]));
            const float own = ptxstd::hsum2(sum), next = __shfl_down_sync(0xffffffffu, own, 1);
            if (f_on && b == 0) p.partial[static_cast<size_t>(rt) * p.W + feature] = own + next;
        }
    }

    // padding of the scale tiles: the CTAs of the first column tile write it
    if (ct == 0) {
        const uint32_t w_rows = static_cast<uint32_t>(mx::padded_rows(p.W));
        if (row0 % 128 == 0)
            for (uint32_t r = p.W + tid; r < w_rows; r += kThreads)
                *reinterpret_cast<uint32_t*>(p.sft + mx::word_offset(r, row0 >> 7, kt)) = 0;
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
    p.wide = (reinterpret_cast<uintptr_t>(p.qt) & 31u) == 0;
    p.col_tiles = (p.cols + kCols - 1) / kCols;
    const uint64_t tiles = p.col_tiles * static_cast<uint64_t>(mx::padded_rows(p.rows) / kRows);
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
    return mx::padded_rows(static_cast<size_t>(rows)) / kRows * static_cast<size_t>(cols) *
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
    r.P = static_cast<uint32_t>(mx::padded_rows(p.rows) / kRows);
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
