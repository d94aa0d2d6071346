// The norms between two blocks of a residual stream, fused with the gate and scale of the joining
// branch and with the quantiser of the next GEMM's operand, and their gradient.
//
// Forward, per row (D columns):
//   p = y ry w_post;  x' = bf16(x + scale g p);  n = x' rx w -> bf16 and / or MX
// It is bound by HBM: x and y are read once, x' and n written once. A row lives in the registers
// of one group of threads between the loads and the stores; the two sums of squares are the only
// exchanges (warp shuffles, then shared memory when a row has more than one warp). x' is rounded to
// bf16 before its norm is taken, because the stored value is what every later reader (the next
// block, the backward pass) sees; n is quantised from f32 without a bf16 step between.
//
// Backward: with a = dn w, the normalised rows h = x' rx and k = y ry, and their means
// m1 = mean(a h), m2 = mean(b k),
//   dx = du + rx (a - h m1),                 dw = sum_rows dn h,
//   dg = scale p dx,  dp = scale g dx,  b = dp w_post,
//   dy = ry (b - k m2),                      dw_post = sum_rows dp k.
// m2 needs dx, hence m1. Substituting dx gives, with t = scale g w_post y,
//   m2 = ry mean(t dx) = ry (sum(t du) + rx (sum(t a) - m1 rx sum(t x'))) / D,  m1 = rx sum(a x') / D,
// so one exchange of four sums serves both means. (No power of rx or ry stands alone: rx^3 leaves
// f32's range for rows around 1e13 or 1e-13, where the norms themselves are still exact.) With one
// gate for all rows both dg and dw_post are column factors times the same sum, S = sum_rows dx y ry:
// dg = scale w_post S, dw_post = scale g S; with a gate per row dg needs no sum and S takes g inside.
// So there are two column sums at most. Each thread keeps its columns for all rows of its group and
// accumulates them in f32; the partial sums go through a workspace and are added in order by a second
// kernel (reproducible, no atomics), which applies the factors.
//
// Both directions are near the issue rate as well as the HBM rate (68 % and 59 % of the issue
// slots, ncu), hence the packed f32 pairs. Forward, 8192 x 8192 with w_post, gate and E4M3 out:
// 472 MB in 77 to 80 us, 6.0 TB/s or 0.92 of the measured copy rate; without w_post in bf16 537 MB
// in 80 us, 1.02 of it; one row of 8192: 3.3 us. Backward, 8192 x 4096: 403 MB in 68 us, 0.91 (72 us
// after a second of load); 2000 x 16384: 393 MB in 137 us, 0.44 (column factors from L2 twice a row).
#include "common.cuh"
#include "data_types.cuh"
#include "mx_block.cuh"
#include "reduce.cuh"

namespace {

namespace dt = ptxstd::data_types;
namespace mx = ptxstd::mx;

using ptxstd::f32x2;
using ptxstd::fma2;
using ptxstd::hsum2;
using ptxstd::mul2;
using ptxstd::narrow;
using ptxstd::Oct;
using ptxstd::pack2f;
using ptxstd::unpack2;
using ptxstd::widen;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Sum over the row's threads: one warp, or the whole block through `red` (32 floats, a buffer of
// its own per call so that one __syncthreads is enough).
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = warp_sum(v);
    if constexpr (WARP_ROW) return v;
    const uint32_t lane = ptxstd::lane_id(), warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < warps ? red[lane] : 0.0f);
}

struct Fwd {
    const uint16_t *x, *y, *w_post, *gate, *w;
    uint16_t *x_out, *n;
    uint8_t *q, *sf;
    float *rstd, *rstd_post;
    float scale, eps;
    uint32_t rows, cols, q_type, blocked;
    size_t gate_stride;  // 0: one gate for all rows
};

// Vector i (eight columns) of a bf16 array. An ordinary load, not ld.global.nc: under programmatic
// launch the kernel before may write the array while this grid is already resident, and a load
// that takes the memory for constant may be moved above the wait or served from an old L1 line.
__device__ __forceinline__ uint4 load16(const uint16_t* p, uint32_t i) {
    return reinterpret_cast<const uint4*>(p)[i];
}

__device__ __forceinline__ f32x2 square_sum(const uint4& v, f32x2 s) {
    const Oct a = widen(v);
#pragma unroll
    for (int k = 0; k < 4; ++k) s = fma2(a.v[k], a.v[k], s);
    return s;
}

// bf16(x + scale gate (y ry w_post)) of eight columns; w_post and gate may be null.
__device__ __forceinline__ uint4 join8(const uint4& xv, const uint4& yv, const uint4* w_post,
                                       const uint4* gate, float ry, float scale) {
    Oct a = widen(yv), x = widen(xv);
    if (w_post) {
        const Oct w = widen(*w_post);
        const f32x2 r = pack2f(ry, ry);
#pragma unroll
        for (int k = 0; k < 4; ++k) a.v[k] = mul2(mul2(a.v[k], r), w.v[k]);
    }
    if (gate) {
        const Oct w = widen(*gate);
#pragma unroll
        for (int k = 0; k < 4; ++k) a.v[k] = mul2(a.v[k], w.v[k]);
    }
    const f32x2 s = pack2f(scale, scale);
#pragma unroll
    for (int k = 0; k < 4; ++k) x.v[k] = fma2(s, a.v[k], x.v[k]);
    return narrow(x);
}

// Where a row's scales go: the scale of vector i (eight columns) at sf[at(i)], written by the first
// of the four lanes that hold a block.
struct ScaleRow {
    uint8_t* sf;
    uint32_t blocked;
    __device__ __forceinline__ ScaleRow(const Fwd& p, uint32_t row, size_t k_tiles)
        : sf(nullptr), blocked(p.blocked) {
        if (p.q)
            sf = p.sf + (blocked ? mx::word_offset(row, 0, k_tiles)
                                 : static_cast<size_t>(row) * (p.cols / 32));
    }
    __device__ __forceinline__ uint32_t at(uint32_t i) const {
        return blocked ? (i >> 4) * 512 + ((i >> 2) & 3u) : i >> 2;
    }
    // The padding columns of a row's last scale tile.
    __device__ __forceinline__ void pad(const Fwd& p, uint32_t tid) const {
        const uint32_t blocks = p.cols / 32;
        if (sf && blocked && tid < 3 && (blocks & 3u) + tid < 4 && (blocks & 3u))
            sf[at(4 * (blocks + tid))] = 0;
    }
};

// n = x' rx w of eight columns (vector i of the row), stored as bf16 and / or quantised. Every
// lane of the warp calls it; lanes outside the row pass on = false and zeros. A block of 32 is the
// vectors of four neighbouring lanes (cols % 32 == 0, so a block is inside the row or outside it
// as a whole).
__device__ __forceinline__ void finish8(const Fwd& p, const uint4& xv, const uint4& wv, float rx,
                                        size_t base, uint32_t i, bool on, uint32_t lane,
                                        const ScaleRow& sr) {
    Oct n = widen(xv);
    const Oct w = widen(wv);
    const f32x2 r = pack2f(rx, rx);
#pragma unroll
    for (int k = 0; k < 4; ++k) n.v[k] = mul2(mul2(n.v[k], r), w.v[k]);
    if (p.n && on) *reinterpret_cast<uint4*>(p.n + base + 8 * i) = narrow(n);
    if (!p.q) return;
    float a[8];
    ptxstd::flatten(n, a);
    const mx::Scale sc = mx::scale_of(mx::amax_quad(mx::amax_of(a)), mx::emax_of(p.q_type));
    if (on) {
        *reinterpret_cast<uint2*>(p.q + base + 8 * i) = mx::pack8(p.q_type, a, sc.inv);
        if ((lane & 3u) == 0) sr.sf[sr.at(i)] = static_cast<uint8_t>(sc.code);
    }
}

// The blocked scales' padding rows: zero.
__device__ __forceinline__ void pad_row(const Fwd& p, uint32_t row, uint32_t tid, uint32_t stride,
                                        size_t k_tiles) {
    if (p.q && p.blocked && row < mx::padded_rows(p.rows))
        for (size_t t = tid; t < k_tiles; t += stride)
            *reinterpret_cast<uint32_t*>(p.sf + mx::word_offset(row, t, k_tiles)) = 0;
}

// scale w_post gate of eight columns (either may be null).
__device__ __forceinline__ Oct branch_factor(const uint16_t* w_post, const uint16_t* gate,
                                             float scale, uint32_t i) {
    Oct f;
#pragma unroll
    for (int k = 0; k < 4; ++k) f.v[k] = pack2f(scale, scale);
    if (w_post) {
        const Oct o = widen(load16(w_post, i));
#pragma unroll
        for (int k = 0; k < 4; ++k) f.v[k] = mul2(f.v[k], o.v[k]);
    }
    if (gate) {
        const Oct o = widen(load16(gate, i));
#pragma unroll
        for (int k = 0; k < 4; ++k) f.v[k] = mul2(f.v[k], o.v[k]);
    }
    return f;
}

// One row per warp or per block, straight from global memory: for few rows (a single row's
// latency), short rows and the longest ones.
constexpr uint32_t kWarpRows = 4;  // rows of a CTA when a warp holds a row

template <int V, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 32 * kWarpRows : 1024)
    norm_kernel(const __grid_constant__ Fwd p) {
    __shared__ float red[2][32];
    const uint32_t lane = ptxstd::lane_id();
    const uint32_t tid = WARP_ROW ? lane : threadIdx.x;
    const uint32_t stride = WARP_ROW ? 32 : blockDim.x;
    const uint32_t row = WARP_ROW ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    const uint32_t nv = p.cols / 8;
    const size_t k_tiles = mx::tiles_k(p.cols / 32);

    ptxstd::pdl_launch_dependents();
    ptxstd::pdl_wait();
    if (row >= p.rows) {
        pad_row(p, row, tid, stride, k_tiles);
        return;
    }
    const size_t base = static_cast<size_t>(row) * p.cols;
    const uint4* const w_post = reinterpret_cast<const uint4*>(p.w_post);
    const uint4* const gate =
        p.gate ? reinterpret_cast<const uint4*>(p.gate + row * p.gate_stride) : nullptr;
    uint4 xv[V], yv[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = tid + j * stride;
        xv[j] = yv[j] = make_uint4(0, 0, 0, 0);
        if (i < nv) {
            xv[j] = *reinterpret_cast<const uint4*>(p.x + base + 8 * i);
            if (p.y) yv[j] = *reinterpret_cast<const uint4*>(p.y + base + 8 * i);
        }
    }
    const float inv_d = 1.0f / static_cast<float>(p.cols);
    if (p.y) {
        float ry = 1.0f;
        if (w_post) {
            f32x2 s = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) s = square_sum(yv[j], s);
            ry = rsqrtf(row_sum<WARP_ROW>(hsum2(s), red[0]) * inv_d + p.eps);
            if (p.rstd_post && tid == 0) p.rstd_post[row] = ry;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
            xv[j] = join8(xv[j], yv[j], w_post ? w_post + i : nullptr, gate ? gate + i : nullptr,
                          ry, p.scale);
            *reinterpret_cast<uint4*>(p.x_out + base + 8 * i) = xv[j];
        }
    }
    f32x2 s = 0;
    uint4 w[V];  // loaded before the exchange, which hides them
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = tid + j * stride;
        w[j] = i < nv ? load16(p.w, i) : make_uint4(0, 0, 0, 0);
        s = square_sum(xv[j], s);
    }
    const float rx = rsqrtf(row_sum<WARP_ROW>(hsum2(s), red[1]) * inv_d + p.eps);
    if (p.rstd && tid == 0) p.rstd[row] = rx;
    const ScaleRow sr(p, row, k_tiles);
    sr.pad(p, tid);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = tid + j * stride;
        finish8(p, xv[j], w[j], rx, base, i, i < nv, lane, sr);
    }
}

// ---- many rows: a ring of rows in shared memory ------------------------------------------------
// One CTA per SM walks the rows blockIdx, blockIdx + grid, ...: its k-th row goes through stage
// k % stages of a ring by bulk copies, and groups of threads take the rows in turn, so that one
// row's sums, another's stores and the loads of later rows overlap. A group copies its row to
// registers first; once it has met in the row's first sum, the stage is free and its first thread
// sends the row `stages` further on into it. The ring is thus in flight nearly all of the time,
// whatever the groups wait for. Column weights sit in shared memory for the CTA's life. The forward
// ring is for rows with both norms (y and w_post given).
constexpr uint32_t kRingBytes = 222 * 1024;
constexpr uint32_t kMaxRing = 12;
enum : uint32_t { kDetailFwd = 0x4200, kDetailBwd = 0x4400 };

__device__ __forceinline__ void group_sync(uint32_t group, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}

struct RingState {
    uint64_t full[kMaxRing];
    uint32_t row[kMaxRing];  // the row whose load is under way in, or has landed in, each stage
    uint32_t abort;
};

// Where row k comes from (the non-null arrays, in this order) and where it goes.
struct Ring {
    RingState& st;
    uint8_t* base;
    const uint16_t* src[5];
    uint32_t arrays, stages, rows, cols;

    __device__ __forceinline__ uint32_t stage_bytes() const { return arrays * cols * 2; }

    __device__ __forceinline__ void init() {
        for (uint32_t i = 0; i < stages; ++i) {
            ptxstd::mbar_init(&st.full[i], 1);
            st.row[i] = ~0u;
        }
        st.abort = 0;
        ptxstd::fence_mbarrier_init();
    }
    // One thread: the CTA's k-th row into `stage`, whose readers are done.
    __device__ __forceinline__ void load(uint32_t k, uint32_t stage) {
        const uint64_t row = blockIdx.x + static_cast<uint64_t>(k) * gridDim.x;
        if (row >= rows) return;
        const uint32_t bytes = cols * 2;
        uint8_t* dst = base + static_cast<size_t>(stage) * stage_bytes();
        ptxstd::mbar_arrive_expect_tx(&st.full[stage], stage_bytes());
#pragma unroll
        for (int i = 0; i < 5; ++i)
            if (src[i]) {
                ptxstd::bulk_load(dst, src[i] + row * cols, bytes, &st.full[stage]);
                dst += bytes;
            }
        *reinterpret_cast<volatile uint32_t*>(&st.row[stage]) = k;
    }
    // Every thread of a group: waits for row k in `stage`. The row number is waited for first: two
    // consecutive rows of a stage may belong to different groups, so a group can be two rows
    // ahead of the stage, where the parity alone would let it pass. Once the number is there, the
    // row before it has been consumed and the barrier is in row k's phase or past it.
    // After a timeout (recorded) the kernel runs on without waiting, on whatever the stages hold,
    // so that every barrier still sees all of its threads; drain() then keeps the block until its
    // copies have landed.
    __device__ __forceinline__ void wait(uint32_t k, uint32_t stage, uint32_t parity, uint32_t* err,
                                         uint32_t detail) {
        volatile uint32_t* abort_flag = &st.abort;
        volatile uint32_t* row = &st.row[stage];
        if (!*abort_flag) {
            bool ok = *row == k;
            if (!ok) {
                const uint64_t t0 = ptxstd::global_timer();
                while (!(ok = *row == k) && !*abort_flag)
                    if (ptxstd::global_timer() - t0 > ptxstd::kWaitLimitNs) break;
            }
            if (!ok || !ptxstd::mbar_wait(&st.full[stage], parity)) {
                ptxstd::record_error(err, PTXSTD_ETIMEOUT, detail | stage);
                *abort_flag = 1u;
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void drain() {
        volatile uint32_t* abort_flag = &st.abort;
        if (!*abort_flag) return;
        const uint32_t mine = rows > blockIdx.x ? (rows - blockIdx.x - 1) / gridDim.x + 1 : 0;
        for (uint32_t i = 0; i < stages && i < mine; ++i) {
            const uint32_t k = *reinterpret_cast<volatile uint32_t*>(&st.row[i]);
            if (k != ~0u) ptxstd::mbar_wait(&st.full[i], (k / stages) & 1u);
        }
    }
};

// Eight f32 column factors per vector in shared memory, the first four columns in one plane and
// the last four in another, so that neighbouring lanes read neighbouring 16 bytes.
__device__ __forceinline__ void store_planes(float4* dst, uint32_t nv, uint32_t i, const Oct& o) {
    const float2 a = unpack2(o.v[0]), b = unpack2(o.v[1]), c = unpack2(o.v[2]),
                 d = unpack2(o.v[3]);
    dst[i] = make_float4(a.x, a.y, b.x, b.y);
    dst[nv + i] = make_float4(c.x, c.y, d.x, d.y);
}
__device__ __forceinline__ Oct load_planes(const float4* src, uint32_t nv, uint32_t i) {
    const float4 a = src[i], b = src[nv + i];
    return {{pack2f(a.x, a.y), pack2f(a.z, a.w), pack2f(b.x, b.y), pack2f(b.z, b.w)}};
}

template <int V, uint32_t THREADS, uint32_t GROUPS>
__global__ void __launch_bounds__(THREADS* GROUPS, 1)
    norm_ring_kernel(const __grid_constant__ Fwd p, uint32_t stages, uint32_t* err) {
    extern __shared__ uint4 ring_smem[];
    __shared__ RingState state;
    constexpr uint32_t kWarps = THREADS / 32;
    __shared__ float4 red[GROUPS][3][kWarps / 4];  // the warps' partial sums; a buffer per exchange
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t nv = p.cols / 8;
    const size_t k_tiles = mx::tiles_k(p.cols / 32);
    const bool gate_rows = p.gate && p.gate_stride;
    // shared memory: w (bf16) | c = scale w_post gate in f32 (the gate of all rows; 1 where there is
    // none) | stages of x | y | gate row
    uint4* const w = ring_smem;
    float4* const c = reinterpret_cast<float4*>(w + nv);
    uint4* const stage0 = w + 3 * nv;
    const uint32_t arrays = 2 + (gate_rows ? 1 : 0);
    Ring ring = {state,
                 reinterpret_cast<uint8_t*>(stage0),
                 {p.x, p.y, gate_rows ? p.gate : nullptr, nullptr, nullptr},
                 arrays, stages, p.rows, p.cols};

    ptxstd::pdl_launch_dependents();
    if (tid == 0) ring.init();
    ptxstd::pdl_wait();
    if (tid == 0)
        for (uint32_t k = 0; k < stages; ++k) ring.load(k, k);
    for (uint32_t i = tid; i < nv; i += blockDim.x) {
        w[i] = load16(p.w, i);
        store_planes(c, nv, i,
                     branch_factor(p.w_post, gate_rows ? nullptr : p.gate, p.scale, i));
    }
    for (uint32_t row = p.rows + blockIdx.x; row < mx::padded_rows(p.rows); row += gridDim.x)
        pad_row(p, row, tid, blockDim.x, k_tiles);
    __syncthreads();

    const uint32_t g = warp / kWarps;
    const uint32_t t = tid - g * THREADS, gw = t >> 5;
    const float inv_d = 1.0f / static_cast<float>(p.cols);
    auto group_sum = [&](float v, float4* buf) {
        v = warp_sum(v);
        if (lane == 0) reinterpret_cast<float*>(buf)[gw] = v;
        group_sync(g, THREADS);
        float4 a = buf[0];
#pragma unroll
        for (uint32_t i = 1; i < kWarps / 4; ++i) {
            const float4 b = buf[i];
            a.x += b.x;
            a.y += b.y;
            a.z += b.z;
            a.w += b.w;
        }
        return (a.x + a.y) + (a.z + a.w);
    };
    uint32_t stage = g % stages, parity = (g / stages) & 1u, flip = 0, k = g;
    for (uint32_t row = blockIdx.x + g * gridDim.x; row < p.rows;
         row += GROUPS * gridDim.x, k += GROUPS) {
        ring.wait(k, stage, parity, err, kDetailFwd);
        const uint4* const xs = stage0 + static_cast<size_t>(stage) * arrays * nv;
        const size_t base = static_cast<size_t>(row) * p.cols;
        uint4 xv[V], yv[V];
        f32x2 s = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = t + j * THREADS;
            xv[j] = yv[j] = make_uint4(0, 0, 0, 0);
            if (i < nv) {
                xv[j] = xs[i];
                yv[j] = xs[nv + i];
            }
            s = square_sum(yv[j], s);
        }
        const float ry = rsqrtf(group_sum(hsum2(s), red[g][0]) * inv_d + p.eps);
        if (t == 0) {
            if (p.rstd_post) p.rstd_post[row] = ry;
            if (!gate_rows) ring.load(k + stages, stage);
        }
        s = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = t + j * THREADS;
            if (i >= nv) continue;
            Oct x = widen(xv[j]), y = widen(yv[j]);
            const Oct f = load_planes(c, nv, i);
            const f32x2 r = pack2f(ry, ry);
            if (gate_rows) {
                const Oct g = widen(xs[2 * nv + i]);
#pragma unroll
                for (int q = 0; q < 4; ++q) y.v[q] = mul2(y.v[q], g.v[q]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) x.v[q] = fma2(mul2(y.v[q], r), f.v[q], x.v[q]);
            xv[j] = narrow(x);
            *reinterpret_cast<uint4*>(p.x_out + base + 8 * i) = xv[j];
            s = square_sum(xv[j], s);
        }
        const float rx = rsqrtf(group_sum(hsum2(s), red[g][1 + flip]) * inv_d + p.eps);
        if (t == 0) {
            if (p.rstd) p.rstd[row] = rx;
            if (gate_rows) ring.load(k + stages, stage);  // the gate row was read until here
        }
        const ScaleRow sr(p, row, k_tiles);
        sr.pad(p, t);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = t + j * THREADS;
            const bool on = i < nv;
            finish8(p, xv[j], on ? w[i] : make_uint4(0, 0, 0, 0), rx, base, i, on, lane, sr);
        }
        flip ^= 1u;
        stage += GROUPS;
        while (stage >= stages) {
            stage -= stages;
            parity ^= 1u;
        }
    }
    ring.drain();
}

template <int V, bool WARP_ROW>
int launch_fwd(const Fwd& p, uint32_t threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const size_t rows = p.q && p.blocked ? mx::padded_rows(p.rows) : p.rows;
    const uint32_t grid = static_cast<uint32_t>(WARP_ROW ? (rows + kWarpRows - 1) / kWarpRows : rows);
    ptxstd::set_pdl(cfg, attr, grid, WARP_ROW ? 32 * kWarpRows : threads, stream);
    if (cudaLaunchKernelEx(&cfg, norm_kernel<V, WARP_ROW>, p) != cudaSuccess) return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

// Stages of a ring of rows beside `fixed` bytes of weights.
uint32_t ring_stages(size_t fixed, size_t row_bytes) {
    if (fixed > kRingBytes) return 0;
    const size_t n = (kRingBytes - fixed) / row_bytes;
    return static_cast<uint32_t>(n < kMaxRing ? n : kMaxRing);
}

template <int V, uint32_t THREADS, uint32_t GROUPS>
int launch_fwd_ring(const Fwd& p, cudaStream_t stream) {
    auto* kernel = norm_ring_kernel<V, THREADS, GROUPS>;
    const size_t vec = static_cast<size_t>(p.cols) * 2, fixed = 3 * vec;
    const size_t row = vec * (2 + (p.gate && p.gate_stride ? 1 : 0));
    // at most 8192 columns: beside 48 KB of weights, three rows of 48 KB; with 4096, eight of 24 KB
    const uint32_t stages = ring_stages(fixed, row);
    if (stages < GROUPS) return PTXSTD_EINVAL;
    const int st = ptxstd::set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes);
    if (st) return st;
    uint32_t* err = ptxstd::device_error_word();
    if (!err) return PTXSTD_ECUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const uint32_t sms = static_cast<uint32_t>(ptxstd::sm_count());
    ptxstd::set_pdl(cfg, attr, p.rows < sms ? p.rows : sms, THREADS * GROUPS, stream);
    cfg.dynamicSmemBytes = fixed + stages * row;
    if (cudaLaunchKernelEx(&cfg, kernel, p, stages, err) != cudaSuccess) return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

// ---- backward ---------------------------------------------------------------------------------
struct Bwd {
    const uint16_t *dn, *du, *x, *w, *y, *w_post, *gate;
    const float *rstd, *rstd_post;
    uint16_t *dx, *dy, *dgate_rows;
    float* partial;  // [groups of the grid][sums][cols]
    float scale;
    uint32_t rows, cols;
    uint32_t sums;  // 1: dw; 2: dw and S
    size_t gate_stride;
};

// Column factors of eight columns: w, and c = scale w_post gate (the gate of all rows; 1 where
// there is none).
struct Factors {
    Oct w, c;
};
__device__ __forceinline__ Factors column_factors(const Bwd& p, uint32_t i) {
    return {widen(load16(p.w, i)),
            branch_factor(p.w_post, p.gate_stride ? nullptr : p.gate, p.scale, i)};
}

// What a row's sums need of eight columns: sum(a x'), sum(t du), sum(t a), sum(t x') with
// a = dn w, t = c gate y. `gate` is this row's own gate, or null.
struct Sums {
    f32x2 ax = 0, td = 0, ta = 0, tx = 0;
};
__device__ __forceinline__ void sums8(Sums& s, const uint4& dnv, const uint4& duv, const uint4& xv,
                                      const uint4& yv, const Factors& f, bool post,
                                      const uint4* gate) {
    Oct a = widen(dnv);
    const Oct x = widen(xv);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        a.v[k] = mul2(a.v[k], f.w.v[k]);
        s.ax = fma2(a.v[k], x.v[k], s.ax);
    }
    if (!post) return;  // without w_post nothing is divided by y's norm
    Oct t = widen(yv);
    const Oct u = widen(duv);
    if (gate) {
        const Oct g = widen(*gate);
#pragma unroll
        for (int k = 0; k < 4; ++k) t.v[k] = mul2(t.v[k], g.v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        t.v[k] = mul2(t.v[k], f.c.v[k]);
        s.td = fma2(t.v[k], u.v[k], s.td);
        s.ta = fma2(t.v[k], a.v[k], s.ta);
        s.tx = fma2(t.v[k], x.v[k], s.tx);
    }
}

// The factors of a row in the gradients, from its sums and statistics.
struct RowFactors {
    float rx, ry, m1, m2;
};
__device__ __forceinline__ RowFactors row_factors(const float4& s, float rx, float ry,
                                                  float inv_d) {
    RowFactors f;
    f.rx = rx;
    f.ry = ry;
    f.m1 = rx * s.x * inv_d;
    f.m2 = ry * (s.y + rx * (s.z - f.m1 * (rx * s.w))) * inv_d;
    return f;
}

// The gradients of eight columns of a row; adds dn x' rx to `dw` and dx y ry (times the row's own
// gate) to `S`.
__device__ __forceinline__ void grads8(const Bwd& p, const RowFactors& r, const uint4& dnv,
                                       const uint4& duv, const uint4& xv, const uint4& yv,
                                       const Factors& f, const uint4* gate, size_t at, Oct& dw,
                                       Oct& S) {
    const Oct dn = widen(dnv), x = widen(xv);
    Oct dx = widen(duv);
    const f32x2 rx = pack2f(r.rx, r.rx), m1 = pack2f(-r.m1, -r.m1);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f32x2 xh = mul2(x.v[k], rx);
        dw.v[k] = fma2(xh, dn.v[k], dw.v[k]);
        dx.v[k] = fma2(rx, fma2(xh, m1, mul2(dn.v[k], f.w.v[k])), dx.v[k]);
    }
    *reinterpret_cast<uint4*>(p.dx + at) = narrow(dx);
    if (!p.y) return;
    Oct y = widen(yv), b;
    const f32x2 ry = pack2f(r.ry, r.ry), m2 = pack2f(-r.m2, -r.m2);
#pragma unroll
    for (int k = 0; k < 4; ++k) y.v[k] = mul2(y.v[k], ry);
#pragma unroll
    for (int k = 0; k < 4; ++k) b.v[k] = mul2(dx.v[k], f.c.v[k]);
    if (gate) {
        const Oct g = widen(*gate);
        Oct dg;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            dg.v[k] = mul2(b.v[k], y.v[k]);
            S.v[k] = fma2(mul2(dx.v[k], g.v[k]), y.v[k], S.v[k]);
            b.v[k] = mul2(b.v[k], g.v[k]);
        }
        *reinterpret_cast<uint4*>(p.dgate_rows + at) = narrow(dg);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) S.v[k] = fma2(dx.v[k], y.v[k], S.v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) b.v[k] = mul2(ry, fma2(y.v[k], m2, b.v[k]));
    *reinterpret_cast<uint4*>(p.dy + at) = narrow(b);
}

__device__ __forceinline__ void store_oct(float* dst, const Oct& o) {
    const float2 a = unpack2(o.v[0]), b = unpack2(o.v[1]), c = unpack2(o.v[2]),
                 d = unpack2(o.v[3]);
    reinterpret_cast<float4*>(dst)[0] = make_float4(a.x, a.y, b.x, b.y);
    reinterpret_cast<float4*>(dst)[1] = make_float4(c.x, c.y, d.x, d.y);
}
__device__ __forceinline__ Oct load_oct(const float* src) {
    const float4 a = reinterpret_cast<const float4*>(src)[0];
    const float4 b = reinterpret_cast<const float4*>(src)[1];
    return {{pack2f(a.x, a.y), pack2f(a.z, a.w), pack2f(b.x, b.y), pack2f(b.z, b.w)}};
}
constexpr Oct kZeroOct = {{0, 0, 0, 0}};

// A warp's four sums, lane 8 q holding sum q (six shuffles: halves of the lanes take halves of the
// sums, then a tree).
__device__ __forceinline__ float warp_sum4(const Sums& q, uint32_t lane) {
    const float4 s = make_float4(hsum2(q.ax), hsum2(q.td), hsum2(q.ta), hsum2(q.tx));
    const bool hi = lane & 16u, odd = lane & 8u;
    float a = hi ? s.z : s.x, b = hi ? s.w : s.y;
    a += __shfl_xor_sync(0xffffffffu, hi ? s.x : s.z, 16);
    b += __shfl_xor_sync(0xffffffffu, hi ? s.y : s.w, 16);
    float c = odd ? b : a;
    c += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int d = 4; d; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
    return c;
}

// Sum over the group's warps: every warp leaves its four sums in buf[warp], every thread adds them
// in warp order. `buf` alternates between rows, so one barrier per row is enough.
template <uint32_t WARPS>
__device__ __forceinline__ float4 group_sum4(const Sums& s, float4* buf, uint32_t warp,
                                             uint32_t lane, uint32_t warps, uint32_t group) {
    const float c = warp_sum4(s, lane);
    if ((lane & 7u) == 0) reinterpret_cast<float*>(buf + warp)[lane >> 3] = c;
    group_sync(group, warps * 32);
    float4 r = buf[0];
#pragma unroll
    for (uint32_t k = 1; k < WARPS; ++k)
        if (k < warps) {
            const float4 o = buf[k];
            r.x += o.x;
            r.y += o.y;
            r.z += o.z;
            r.w += o.w;
        }
    return r;
}

// Rows of up to 1024 columns (few threads per row, many blocks per SM) and of more than 8192 (whose
// column sums need shared memory). V vectors per thread.
template <int V>
__global__ void __launch_bounds__(V == 1 ? 128 : 512)
    norm_backward_kernel(const __grid_constant__ Bwd p) {
    constexpr bool kShared = V > 1;
    constexpr uint32_t kMaxWarps = V == 1 ? 4 : 16;
    extern __shared__ float acc_smem[];  // [sums][cols] when kShared
    __shared__ float4 red[2][kMaxWarps];
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t warps = blockDim.x >> 5, stride = blockDim.x, nv = p.cols / 8;
    Oct dw = kZeroOct, S = kZeroOct;
    ptxstd::pdl_launch_dependents();
    if constexpr (kShared) {
        for (uint32_t i = tid; i < p.sums * p.cols; i += stride) acc_smem[i] = 0.0f;
        __syncthreads();
    }
    ptxstd::pdl_wait();

    const float inv_d = 1.0f / static_cast<float>(p.cols);
    uint32_t flip = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1u) {
        const size_t base = static_cast<size_t>(row) * p.cols;
        const uint4* const gate =
            p.gate_stride ? reinterpret_cast<const uint4*>(p.gate + base) : nullptr;
        uint4 dnv[V], duv[V], xv[V], yv[V];
        Sums s;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            dnv[j] = duv[j] = xv[j] = yv[j] = make_uint4(0, 0, 0, 0);
            if (i < nv) {
                dnv[j] = *reinterpret_cast<const uint4*>(p.dn + base + 8 * i);
                xv[j] = *reinterpret_cast<const uint4*>(p.x + base + 8 * i);
                if (p.du) duv[j] = *reinterpret_cast<const uint4*>(p.du + base + 8 * i);
                if (p.y) yv[j] = *reinterpret_cast<const uint4*>(p.y + base + 8 * i);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i < nv)
                sums8(s, dnv[j], duv[j], xv[j], yv[j], column_factors(p, i), p.w_post,
                      gate ? gate + i : nullptr);
        }
        const float4 sum = group_sum4<kMaxWarps>(s, red[flip], warp, lane, warps, 0);
        const RowFactors r =
            row_factors(sum, p.rstd[row], p.w_post ? p.rstd_post[row] : 1.0f, inv_d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
            if constexpr (kShared) {
                float *a = acc_smem + 8 * i, *b = a + p.cols;
                dw = load_oct(a);
                if (p.sums > 1) S = load_oct(b);
                grads8(p, r, dnv[j], duv[j], xv[j], yv[j], column_factors(p, i),
                       gate ? gate + i : nullptr, base + 8 * i, dw, S);
                store_oct(a, dw);
                if (p.sums > 1) store_oct(b, S);
            } else {
                grads8(p, r, dnv[j], duv[j], xv[j], yv[j], column_factors(p, i),
                       gate ? gate + i : nullptr, base + 8 * i, dw, S);
            }
        }
    }
    float* out = p.partial + static_cast<size_t>(blockIdx.x) * p.sums * p.cols;
    if constexpr (kShared) {
        __syncthreads();
        for (uint32_t i = tid; i < p.sums * p.cols; i += stride) out[i] = acc_smem[i];
    } else if (tid < nv) {
        store_oct(out + 8 * tid, dw);
        if (p.sums > 1) store_oct(out + p.cols + 8 * tid, S);
    }
}

// 1024 < columns <= 8192: the ring. GROUPS groups of THREADS threads take the CTA's rows in turn;
// a thread keeps its V vectors' column sums in registers for all of its group's rows.
template <int V, uint32_t THREADS, uint32_t GROUPS>
__global__ void __launch_bounds__(THREADS* GROUPS, 1)
    norm_backward_ring_kernel(const __grid_constant__ Bwd p, uint32_t stages, uint32_t* err) {
    constexpr uint32_t kWarps = THREADS / 32;
    extern __shared__ uint4 ring_smem[];
    __shared__ RingState state;
    __shared__ float4 red[GROUPS][2][kWarps];
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t nv = p.cols / 8;
    // shared memory: column factors w | c in f32, stages of dn | x | du | y | gate row
    float4* const w = reinterpret_cast<float4*>(ring_smem);
    float4* const c = w + 2 * nv;
    uint4* const stage0 = ring_smem + 4 * nv;
    const uint32_t arrays = 2 + (p.du ? 1 : 0) + (p.y ? 1 : 0) + (p.gate_stride ? 1 : 0);
    Ring ring = {state,
                 reinterpret_cast<uint8_t*>(stage0),
                 {p.dn, p.x, p.du, p.y, p.gate_stride ? p.gate : nullptr},
                 arrays, stages, p.rows, p.cols};

    ptxstd::pdl_launch_dependents();
    if (tid == 0) ring.init();
    ptxstd::pdl_wait();
    if (tid == 0)
        for (uint32_t k = 0; k < stages; ++k) ring.load(k, k);
    for (uint32_t i = tid; i < nv; i += blockDim.x) {
        const Factors f = column_factors(p, i);
        store_planes(w, nv, i, f.w);
        store_planes(c, nv, i, f.c);
    }
    __syncthreads();

    const uint32_t g = warp / kWarps;
    const uint32_t t = tid - g * THREADS, gw = t >> 5;
    const float inv_d = 1.0f / static_cast<float>(p.cols);
    Oct dw[V], S[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[j] = S[j] = kZeroOct;
    uint32_t stage = g % stages, parity = (g / stages) & 1u, flip = 0, k = g;
    for (uint32_t row = blockIdx.x + g * gridDim.x; row < p.rows;
         row += GROUPS * gridDim.x, k += GROUPS, flip ^= 1u) {
        const float rx = p.rstd[row], ry = p.w_post ? p.rstd_post[row] : 1.0f;
        ring.wait(k, stage, parity, err, kDetailBwd);
        const uint4* const dns = stage0 + static_cast<size_t>(stage) * arrays * nv;
        const uint4* const xs = dns + nv;
        const uint4* const dus = xs + nv;
        const uint4* const ys = dus + (p.du ? nv : 0);
        const uint4* const gs = p.gate_stride ? ys + nv : nullptr;
        uint4 dnv[V], duv[V], xv[V], yv[V];
        Sums s;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = t + j * THREADS;
            dnv[j] = duv[j] = xv[j] = yv[j] = make_uint4(0, 0, 0, 0);
            if (i < nv) {
                dnv[j] = dns[i];
                xv[j] = xs[i];
                if (p.du) duv[j] = dus[i];
                if (p.y) yv[j] = ys[i];
                sums8(s, dnv[j], duv[j], xv[j], yv[j], {load_planes(w, nv, i), load_planes(c, nv, i)},
                      p.w_post, gs ? gs + i : nullptr);
            }
        }
        const float4 sum = group_sum4<kWarps>(s, red[g][flip], gw, lane, kWarps, g);
        if (t == 0 && !gs) ring.load(k + stages, stage);
        const RowFactors r = row_factors(sum, rx, ry, inv_d);
        const size_t base = static_cast<size_t>(row) * p.cols;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = t + j * THREADS;
            if (i < nv)
                grads8(p, r, dnv[j], duv[j], xv[j], yv[j],
                       {load_planes(w, nv, i), load_planes(c, nv, i)}, gs ? gs + i : nullptr,
                       base + 8 * i, dw[j], S[j]);
        }
        if (gs) {  // the gate row was read until here
            group_sync(g, THREADS);
            if (t == 0) ring.load(k + stages, stage);
        }
        stage += GROUPS;
        while (stage >= stages) {
            stage -= stages;
            parity ^= 1u;
        }
    }
    float* out = p.partial + static_cast<size_t>(blockIdx.x * GROUPS + g) * p.sums * p.cols;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = t + j * THREADS;
        if (i >= nv) continue;
        store_oct(out + 8 * i, dw[j]);
        if (p.sums > 1) store_oct(out + p.cols + 8 * i, S[j]);
    }
    ring.drain();
}

// How a backward call runs, by its sizes: the grid and the groups that write partial sums.
struct BwdPlan {
    bool ring;
    uint32_t grid, groups;
};
BwdPlan bwd_plan(int64_t rows, int64_t cols) {
    const int64_t sms = ptxstd::sm_count();
    BwdPlan b = {};
    b.ring = cols > 1024 && cols <= 8192;
    b.groups = b.ring && cols <= 4096 ? 2 : 1;
    const int64_t grid = cols <= 1024 ? 8 * sms : sms;  // 128-thread blocks: eight per SM
    b.grid = static_cast<uint32_t>(rows < grid ? rows : grid);
    return b;
}

template <int V>
int launch_bwd(const Bwd& p, uint32_t grid, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    const uint32_t nv = p.cols / 8;
    ptxstd::set_pdl(cfg, attr, grid, ((nv + V - 1) / V + 31) / 32 * 32, stream);
    if (V > 1) {
        cfg.dynamicSmemBytes = static_cast<size_t>(p.sums) * p.cols * 4;
        const int st = ptxstd::set_max_dynamic_smem(
            reinterpret_cast<const void*>(norm_backward_kernel<V>), 2 * 16384 * 4);
        if (st) return st;
    }
    if (cudaLaunchKernelEx(&cfg, norm_backward_kernel<V>, p) != cudaSuccess) return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

template <int V, uint32_t THREADS, uint32_t GROUPS>
int launch_bwd_ring(const Bwd& p, uint32_t grid, cudaStream_t stream) {
    auto* kernel = norm_backward_ring_kernel<V, THREADS, GROUPS>;
    const int st = ptxstd::set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes);
    if (st) return st;
    uint32_t* err = ptxstd::device_error_word();
    if (!err) return PTXSTD_ECUDA;
    const size_t vec = static_cast<size_t>(p.cols) * 2, fixed = 4 * vec;
    const size_t row = vec * (2 + (p.du ? 1 : 0) + (p.y ? 1 : 0) + (p.gate_stride ? 1 : 0));
    // at most 8192 columns: beside 64 KB of factors, two rows of 64 KB or one of 80 KB
    const uint32_t stages = ring_stages(fixed, row);
    if (stages < GROUPS) return PTXSTD_EINVAL;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    ptxstd::set_pdl(cfg, attr, grid, THREADS * GROUPS, stream);
    cfg.dynamicSmemBytes = fixed + stages * row;
    if (cudaLaunchKernelEx(&cfg, kernel, p, stages, err) != cudaSuccess) return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

bool misaligned(const void* p) { return p && !ptxstd::aligned16(p); }

}  // namespace

extern "C" int ptxstd_rmsnorm_residual(const uint16_t* d_x, const uint16_t* d_y,
                                       const uint16_t* d_w_post, const uint16_t* d_gate,
                                       int64_t gate_rows, float scale, const uint16_t* d_w,
                                       float eps, int64_t rows, int64_t cols, uint16_t* d_x_out,
                                       uint16_t* d_n, int out_type, uint8_t* d_q, uint8_t* d_sf,
                                       int sf_layout, float* d_rstd, float* d_rstd_post,
                                       ptxstd_stream stream) {
    if (rows <= 0 || cols <= 0 || cols % 8 || cols > 32768 || rows >= (1ll << 31) - 128)
        return PTXSTD_EINVAL;
    if (!(eps >= 0.0f)) return PTXSTD_EINVAL;
    if (!d_x || !d_w || (!d_n && !d_q)) return PTXSTD_EINVAL;
    if ((d_y != nullptr) != (d_x_out != nullptr)) return PTXSTD_EINVAL;
    if (!d_y && (d_w_post || d_gate || d_rstd_post)) return PTXSTD_EINVAL;
    if (d_rstd_post && !d_w_post) return PTXSTD_EINVAL;
    if (d_gate && gate_rows != 1 && gate_rows != rows) return PTXSTD_EINVAL;
    if (d_q) {
        if (!d_sf || cols % 32 || (sf_layout != 0 && sf_layout != 1)) return PTXSTD_EINVAL;
        if (out_type != PTXSTD_MX_E4M3 && out_type != PTXSTD_MX_E5M2) return PTXSTD_EINVAL;
    }
    if (misaligned(d_x) || misaligned(d_y) || misaligned(d_w_post) || misaligned(d_gate) ||
        misaligned(d_w) || misaligned(d_x_out) || misaligned(d_n) || misaligned(d_q) ||
        misaligned(d_sf) || misaligned(d_rstd) || misaligned(d_rstd_post))
        return PTXSTD_EINVAL;
    Fwd p = {};
    p.x = d_x;
    p.y = d_y;
    p.w_post = d_w_post;
    p.gate = d_gate;
    p.w = d_w;
    p.x_out = d_x_out;
    p.n = d_n;
    p.q = d_q;
    p.sf = d_sf;
    p.rstd = d_rstd;
    p.rstd_post = d_rstd_post;
    p.scale = scale;
    p.eps = eps;
    p.rows = static_cast<uint32_t>(rows);
    p.cols = static_cast<uint32_t>(cols);
    p.q_type = static_cast<uint32_t>(out_type);
    p.blocked = static_cast<uint32_t>(sf_layout);
    p.gate_stride = gate_rows == 1 ? 0 : static_cast<size_t>(cols);
    auto s = static_cast<cudaStream_t>(stream);
    const uint32_t nv = p.cols / 8;
    if (nv <= 32) return launch_fwd<1, true>(p, 32, s);
    if (nv <= 64) return launch_fwd<2, true>(p, 32, s);
    if (nv <= 128) return launch_fwd<4, true>(p, 32, s);
    // The ring pays where a row has two exchanges and there is enough to stream: with w_post,
    // gate, E4M3 out, 8192 x 8192 takes 77 to 80 us against 92 us for a row per block, 8192 x 4096
    // 42.0 against 47.1 us, 8192 x 2048 25.8 against 30.0 us, 6000 x 2048 19.9 against 23.1 us. Below
    // the limit the two come together (4000 x 2048 15.3 against 16.8 us, 2400 x 4096 17.3 against
    // 17.7 us, 1200 x 8192 18.3 against 18.7 us), and a row per block is the faster one for rows that
    // leave much of the long rows' groups idle (3000 x 5152: 26.9 us, the ring 28.1 us). Without
    // w_post it is at the copy rate already (8192 x 8192 in bf16: 80 us).
    if (d_w_post && rows * cols >= 12'000'000) {
        if (nv <= 256) return launch_fwd_ring<2, 128, 6>(p, s);
        if (nv <= 512) return launch_fwd_ring<4, 128, 6>(p, s);
        if (nv > 768 && nv <= 1024) return launch_fwd_ring<4, 256, 3>(p, s);
    }
    // A row per block: one vector per thread while a block can be that large and a row's latency
    // counts (100 x 4096: 3.4 us, 3.8 us with two); two once an SM has several rows, so that more
    // blocks fit (300 x 8192 6.2 against 7.6 us, 1200 x 4096 8.8 against 10.4 us), but for a gate
    // per row, whose third stream keeps enough loads in flight (1037 x 5152 10.2 against 11.1 us).
    const bool few = rows <= ptxstd::sm_count() || (d_gate && p.gate_stride);
    const int v = nv > 2048 ? 4 : nv > 1024 || (nv > 256 && !few) ? 2 : 1;
    const uint32_t threads = ((nv + v - 1) / v + 31) / 32 * 32;
    if (v == 1) return launch_fwd<1, false>(p, threads, s);
    if (v == 2) return launch_fwd<2, false>(p, threads, s);
    return launch_fwd<4, false>(p, threads, s);
}

extern "C" size_t ptxstd_rmsnorm_residual_backward_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols % 8 || cols > 16384) return 0;
    const BwdPlan b = bwd_plan(rows, cols);
    return static_cast<size_t>(b.grid) * b.groups * 2 * static_cast<size_t>(cols) * 4;
}

extern "C" int ptxstd_rmsnorm_residual_backward(
    const uint16_t* d_dn, const uint16_t* d_dx_out, const uint16_t* d_x_out, const uint16_t* d_w,
    const float* d_rstd, const uint16_t* d_y, const uint16_t* d_w_post, const float* d_rstd_post,
    const uint16_t* d_gate, int64_t gate_rows, float scale, int64_t rows, int64_t cols,
    uint16_t* d_dx, float* d_dw, uint16_t* d_dy, float* d_dw_post, void* d_dgate,
    void* d_workspace, size_t workspace_bytes, ptxstd_stream stream) {
    if (rows <= 0 || cols <= 0 || cols % 8 || cols > 16384 || rows >= (1ll << 31) - 128)
        return PTXSTD_EINVAL;
    if (!d_dn || !d_x_out || !d_w || !d_rstd || !d_dx || !d_dw || !d_workspace)
        return PTXSTD_EINVAL;
    if (!d_y && (d_w_post || d_gate || d_rstd_post)) return PTXSTD_EINVAL;
    if ((d_y != nullptr) != (d_dy != nullptr)) return PTXSTD_EINVAL;
    if ((d_w_post != nullptr) != (d_rstd_post != nullptr) ||
        (d_w_post != nullptr) != (d_dw_post != nullptr) ||
        (d_gate != nullptr) != (d_dgate != nullptr))
        return PTXSTD_EINVAL;
    if (d_gate && gate_rows != 1 && gate_rows != rows) return PTXSTD_EINVAL;
    if (misaligned(d_dn) || misaligned(d_dx_out) || misaligned(d_x_out) || misaligned(d_w) ||
        misaligned(d_rstd) || misaligned(d_y) || misaligned(d_w_post) || misaligned(d_rstd_post) ||
        misaligned(d_gate) || misaligned(d_dx) || misaligned(d_dw) || misaligned(d_dy) ||
        misaligned(d_dw_post) || misaligned(d_dgate) || misaligned(d_workspace))
        return PTXSTD_EINVAL;
    if (workspace_bytes < ptxstd_rmsnorm_residual_backward_workspace_bytes(rows, cols))
        return PTXSTD_EINVAL;
    const BwdPlan plan = bwd_plan(rows, cols);
    Bwd p = {};
    p.dn = d_dn;
    p.du = d_dx_out;
    p.x = d_x_out;
    p.w = d_w;
    p.y = d_y;
    p.w_post = d_w_post;
    p.gate = d_gate;
    p.rstd = d_rstd;
    p.rstd_post = d_rstd_post;
    p.dx = d_dx;
    p.dy = d_dy;
    p.scale = scale;
    p.rows = static_cast<uint32_t>(rows);
    p.cols = static_cast<uint32_t>(cols);
    // a single row's gate is a gate of all rows either way: its gradient is f32 [cols]
    const bool vector_gate = d_gate && gate_rows == 1;
    if (d_gate && !vector_gate) {
        p.dgate_rows = static_cast<uint16_t*>(d_dgate);
        p.gate_stride = static_cast<size_t>(cols);
    }
    p.sums = d_w_post || vector_gate ? 2 : 1;
    p.partial = static_cast<float*>(d_workspace);
    auto s = static_cast<cudaStream_t>(stream);
    int st;
    if (!plan.ring)
        st = cols <= 1024 ? launch_bwd<1>(p, plan.grid, s) : launch_bwd<4>(p, plan.grid, s);
    else if (cols <= 2048)
        st = launch_bwd_ring<1, 256, 2>(p, plan.grid, s);
    else if (cols <= 4096)
        st = launch_bwd_ring<2, 256, 2>(p, plan.grid, s);
    else
        st = launch_bwd_ring<2, 512, 1>(p, plan.grid, s);
    if (st) return st;
    ptxstd::Reduce r = {};
    r.partial = p.partial;
    r.P = plan.grid * plan.groups;
    r.sums = p.sums;
    r.cols = p.cols;
    r.scale = scale;
    r.o0 = d_dw;
    r.o1 = d_dw_post;
    r.f1 = vector_gate ? d_gate : nullptr;
    r.o2 = vector_gate ? static_cast<float*>(d_dgate) : nullptr;
    r.f2 = d_w_post;
    return ptxstd::launch_reduce(r, s);
}
