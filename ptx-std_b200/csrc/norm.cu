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
// Backward: with a = dn w,
//   dx = du + rx a - x' rx^3 mean(a x'),   dw = sum_rows dn x' rx,
//   dg = scale p dx,  dp = scale g dx,  b = dp w_post,
//   dy = ry b - y ry^3 mean(b y),          dw_post = sum_rows dp y ry.
// mean(b y) needs dx, hence mean(a x'). Substituting dx gives, with t = scale g w_post y,
//   sum(b y) = sum(t du) + rx sum(t a) - (rx^3 mean(a x')) sum(t x'),
// so one exchange of four sums serves both means. Each thread keeps its columns for all rows of
// the CTA and accumulates the column sums in f32 registers; the CTAs' partial sums go through a
// workspace and are added in CTA order by a second kernel (reproducible, no atomics).
#include "common.cuh"
#include "data_types.cuh"
#include "mx_block.cuh"
#include "reduce.cuh"

namespace {

namespace dt = ptxstd::data_types;
namespace mx = ptxstd::mx;

__device__ __forceinline__ void unpack8(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        o[2 * k] = dt::bf16_lo(w[k]);
        o[2 * k + 1] = dt::bf16_hi(w[k]);
    }
}
__device__ __forceinline__ uint4 pack8(const float (&o)[8]) {
    return make_uint4(dt::bf16x2_from_f32(o[0], o[1]), dt::bf16x2_from_f32(o[2], o[3]),
                      dt::bf16x2_from_f32(o[4], o[5]), dt::bf16x2_from_f32(o[6], o[7]));
}
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
    if (row >= p.rows) {  // padding rows of the blocked scales
        if (p.q && p.blocked && row < mx::padded_rows(p.rows))
            for (size_t t = tid; t < k_tiles; t += stride)
                *reinterpret_cast<uint32_t*>(p.sf + mx::word_offset(row, t, k_tiles)) = 0;
        return;
    }
    const size_t base = static_cast<size_t>(row) * p.cols;
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
        if (p.w_post) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float a[8];
                unpack8(yv[j], a);
#pragma unroll
                for (int k = 0; k < 8; ++k) s = fmaf(a[k], a[k], s);
            }
            ry = rsqrtf(row_sum<WARP_ROW>(s, red[0]) * inv_d + p.eps);
            if (p.rstd_post && tid == 0) p.rstd_post[row] = ry;
        }
        const uint16_t* gate = p.gate ? p.gate + row * p.gate_stride : nullptr;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
            float a[8], x[8], w[8];
            unpack8(yv[j], a);
            unpack8(xv[j], x);
            if (p.w_post) {
                unpack8(__ldg(reinterpret_cast<const uint4*>(p.w_post + 8 * i)), w);
#pragma unroll
                for (int k = 0; k < 8; ++k) a[k] = a[k] * ry * w[k];
            }
            if (gate) {
                unpack8(__ldg(reinterpret_cast<const uint4*>(gate + 8 * i)), w);
#pragma unroll
                for (int k = 0; k < 8; ++k) a[k] *= w[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = fmaf(p.scale, a[k], x[k]);
            xv[j] = pack8(x);
            *reinterpret_cast<uint4*>(p.x_out + base + 8 * i) = xv[j];
        }
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float a[8];
        unpack8(xv[j], a);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fmaf(a[k], a[k], s);
    }
    const float rx = rsqrtf(row_sum<WARP_ROW>(s, red[1]) * inv_d + p.eps);
    if (p.rstd && tid == 0) p.rstd[row] = rx;
    const uint32_t emax = mx::emax_of(p.q_type);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = tid + j * stride;
        const bool on = i < nv;
        float a[8], w[8];
        unpack8(xv[j], a);
        unpack8(on ? __ldg(reinterpret_cast<const uint4*>(p.w + 8 * i)) : make_uint4(0, 0, 0, 0),
                w);
#pragma unroll
        for (int k = 0; k < 8; ++k) a[k] = a[k] * rx * w[k];
        if (p.n && on) *reinterpret_cast<uint4*>(p.n + base + 8 * i) = pack8(a);
        if (p.q) {
            // a block of 32 is the vectors of four neighbouring lanes (cols % 32 == 0, so a block
            // is inside the row or outside it as a whole); lanes outside hold zeros
            const float m = mx::amax_quad(mx::amax_of(a));  // every lane takes part
            const uint32_t code = on ? mx::scale_code(m, emax) : 0u;
            const float inv = dt::ue8m0_inverse(code);
            if (on)
                *reinterpret_cast<uint2*>(p.q + base + 8 * i) =
                    make_uint2(mx::pack4(p.q_type, a[0], a[1], a[2], a[3], inv),
                               mx::pack4(p.q_type, a[4], a[5], a[6], a[7], inv));
            if (p.blocked) {
                // four blocks' codes (16 lanes) as one word of the scale tile
                uint32_t c = code | __shfl_down_sync(0xffffffffu, code, 4) << 8;
                c |= __shfl_down_sync(0xffffffffu, c, 8) << 16;
                if ((lane & 15u) == 0 && on)
                    *reinterpret_cast<uint32_t*>(p.sf + mx::word_offset(row, i >> 4, k_tiles)) = c;
            } else if ((lane & 3u) == 0 && on) {
                p.sf[static_cast<size_t>(row) * (p.cols / 32) + (i >> 2)] =
                    static_cast<uint8_t>(code);
            }
        }
    }
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

// ---- backward ---------------------------------------------------------------------------------
struct Bwd {
    const uint16_t *dn, *du, *x, *w, *y, *w_post, *gate;
    const float *rstd, *rstd_post;
    uint16_t *dx, *dy, *dgate_rows;
    float* partial;  // [grid][sums][cols]
    float scale;
    uint32_t rows, cols;
    uint32_t sums;      // 1 dw, + dw_post, + dgate (vector gate), in that order
    uint32_t post_at, gate_at;  // index of their sums, or 0
    size_t gate_stride;
};

// Column sums of a thread's V vectors, in registers, or in shared memory when V is large.
template <int V>
__global__ void __launch_bounds__(V == 4 ? 512 : 512)
    norm_backward_kernel(const __grid_constant__ Bwd p) {
    constexpr bool kShared = V == 4;
    extern __shared__ float acc_smem[];  // [3][cols] when kShared
    __shared__ float red[2][4][16];
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id(), warp = tid >> 5;
    const uint32_t warps = blockDim.x >> 5, stride = blockDim.x, nv = p.cols / 8;
    float acc[kShared ? 1 : 3][kShared ? 1 : V][8];
    ptxstd::pdl_launch_dependents();
    if constexpr (kShared) {
        for (uint32_t i = tid; i < p.sums * p.cols; i += stride) acc_smem[i] = 0.0f;
        __syncthreads();
    } else {
#pragma unroll
        for (int s = 0; s < 3; ++s)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[s][j][k] = 0.0f;
    }
    auto add = [&](uint32_t s, int si, int j, uint32_t i, const float (&v)[8]) {
        if constexpr (kShared) {
            float4* a = reinterpret_cast<float4*>(acc_smem + s * p.cols + 8 * i);
            float4 lo = a[0], hi = a[1];
            lo.x += v[0]; lo.y += v[1]; lo.z += v[2]; lo.w += v[3];
            hi.x += v[4]; hi.y += v[5]; hi.z += v[6]; hi.w += v[7];
            a[0] = lo;
            a[1] = hi;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[si][j][k] += v[k];
        }
    };
    ptxstd::pdl_wait();

    const float inv_d = 1.0f / static_cast<float>(p.cols);
    uint32_t flip = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, flip ^= 1u) {
        const size_t base = static_cast<size_t>(row) * p.cols;
        const uint16_t* gate = p.gate ? p.gate + row * p.gate_stride : nullptr;
        uint4 dnv[V], duv[V], xv[V], yv[V];
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
        const float rx = p.rstd[row];
        const float ry = p.w_post ? p.rstd_post[row] : 1.0f;
        float s_ax = 0.0f, s_td = 0.0f, s_ta = 0.0f, s_tx = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
            float dn[8], x[8], w[8];
            unpack8(dnv[j], dn);
            unpack8(xv[j], x);
            unpack8(__ldg(reinterpret_cast<const uint4*>(p.w + 8 * i)), w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                dn[k] *= w[k];
                s_ax = fmaf(dn[k], x[k], s_ax);
            }
            if (p.w_post) {
                float t[8], u[8];
                unpack8(yv[j], t);
                unpack8(__ldg(reinterpret_cast<const uint4*>(p.w_post + 8 * i)), u);
#pragma unroll
                for (int k = 0; k < 8; ++k) t[k] *= p.scale * u[k];
                if (gate) {
                    unpack8(__ldg(reinterpret_cast<const uint4*>(gate + 8 * i)), u);
#pragma unroll
                    for (int k = 0; k < 8; ++k) t[k] *= u[k];
                }
                unpack8(duv[j], u);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    s_td = fmaf(t[k], u[k], s_td);
                    s_ta = fmaf(t[k], dn[k], s_ta);
                    s_tx = fmaf(t[k], x[k], s_tx);
                }
            }
        }
        s_ax = warp_sum(s_ax);
        if (p.w_post) {
            s_td = warp_sum(s_td);
            s_ta = warp_sum(s_ta);
            s_tx = warp_sum(s_tx);
        }
        if (lane == 0) {
            red[flip][0][warp] = s_ax;
            red[flip][1][warp] = s_td;
            red[flip][2][warp] = s_ta;
            red[flip][3][warp] = s_tx;
        }
        __syncthreads();  // one per row: the two halves of `red` alternate
        s_ax = warp_sum(lane < warps ? red[flip][0][lane & 15] : 0.0f);
        const float k1 = rx * rx * rx * (s_ax * inv_d);
        float k2 = 0.0f;
        if (p.w_post) {
            s_td = warp_sum(lane < warps ? red[flip][1][lane & 15] : 0.0f);
            s_ta = warp_sum(lane < warps ? red[flip][2][lane & 15] : 0.0f);
            s_tx = warp_sum(lane < warps ? red[flip][3][lane & 15] : 0.0f);
            k2 = ry * ry * ry * ((s_td + rx * s_ta - k1 * s_tx) * inv_d);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
            float dx[8], x[8], dn[8], w[8], v[8];
            unpack8(dnv[j], dn);
            unpack8(xv[j], x);
            unpack8(duv[j], dx);
            unpack8(__ldg(reinterpret_cast<const uint4*>(p.w + 8 * i)), w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = dn[k] * x[k] * rx;
                dx[k] += rx * (dn[k] * w[k]) - x[k] * k1;
            }
            add(0, 0, j, i, v);
            *reinterpret_cast<uint4*>(p.dx + base + 8 * i) = pack8(dx);
            if (p.y) {
                float y[8], g[8], wp[8];
                unpack8(yv[j], y);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    dx[k] *= p.scale;
                    g[k] = wp[k] = 1.0f;
                }
                if (p.w_post) unpack8(__ldg(reinterpret_cast<const uint4*>(p.w_post + 8 * i)), wp);
                if (gate) {
                    unpack8(__ldg(reinterpret_cast<const uint4*>(gate + 8 * i)), g);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = dx[k] * (y[k] * ry * wp[k]);
                    if (p.dgate_rows)
                        *reinterpret_cast<uint4*>(p.dgate_rows + base + 8 * i) = pack8(v);
                    else
                        add(p.gate_at, 2, j, i, v);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) dx[k] *= g[k];  // dp
                if (p.w_post) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = dx[k] * y[k] * ry;
                    add(p.post_at, 1, j, i, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) dx[k] = ry * (dx[k] * wp[k]) - y[k] * k2;
                }
                *reinterpret_cast<uint4*>(p.dy + base + 8 * i) = pack8(dx);
            }
        }
    }
    float* out = p.partial + static_cast<size_t>(blockIdx.x) * p.sums * p.cols;
    if constexpr (kShared) {
        __syncthreads();
        for (uint32_t i = tid; i < p.sums * p.cols; i += stride) out[i] = acc_smem[i];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t i = tid + j * stride;
            if (i >= nv) continue;
#pragma unroll
            for (int s = 0; s < 3; ++s) {
                const uint32_t at = s == 0 ? 0 : s == 1 ? p.post_at : p.gate_at;
                if (s > 0 && at == 0) continue;
                float4* o = reinterpret_cast<float4*>(out + at * p.cols + 8 * i);
                o[0] = make_float4(acc[s][j][0], acc[s][j][1], acc[s][j][2], acc[s][j][3]);
                o[1] = make_float4(acc[s][j][4], acc[s][j][5], acc[s][j][6], acc[s][j][7]);
            }
        }
    }
}

// CTAs of the backward kernel: its threads hold V vectors each.
int bwd_vectors(int64_t cols) { return cols <= 4096 ? 1 : cols <= 8192 ? 2 : 4; }
uint32_t bwd_threads(int64_t cols) {
    const int64_t v = bwd_vectors(cols), nv = cols / 8;
    return static_cast<uint32_t>(((nv + v - 1) / v + 31) / 32 * 32);
}
int64_t bwd_grid(int64_t rows, int64_t cols) {
    const int64_t per_sm = cols > 8192 ? 1 : 1024 / bwd_threads(cols) > 8 ? 8 : 1024 / bwd_threads(cols);
    const int64_t g = static_cast<int64_t>(ptxstd::sm_count()) * per_sm;
    return rows < g ? rows : g;
}

template <int V>
int launch_bwd(const Bwd& p, uint32_t grid, uint32_t threads, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    ptxstd::set_pdl(cfg, attr, grid, threads, stream);
    if (V == 4) {
        cfg.dynamicSmemBytes = static_cast<size_t>(p.sums) * p.cols * 4;
        const int st = ptxstd::set_max_dynamic_smem(
            reinterpret_cast<const void*>(norm_backward_kernel<V>), 3 * 16384 * 4);
        if (st) return st;
    }
    if (cudaLaunchKernelEx(&cfg, norm_backward_kernel<V>, p) != cudaSuccess) return PTXSTD_ECUDA;
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
    // few rows: one vector per thread (the row's latency counts); many rows: four (fewer threads
    // per row, more loads in flight per thread)
    const int v = nv > 2048 || rows > 296 ? 4 : nv > 1024 ? 2 : 1;
    const uint32_t threads = ((nv + v - 1) / v + 31) / 32 * 32;
    if (v == 1) return launch_fwd<1, false>(p, threads, s);
    if (v == 2) return launch_fwd<2, false>(p, threads, s);
    return launch_fwd<4, false>(p, threads, s);
}

extern "C" size_t ptxstd_rmsnorm_residual_backward_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols % 8 || cols > 16384) return 0;
    return static_cast<size_t>(bwd_grid(rows, cols)) * 3 * static_cast<size_t>(cols) * 4;
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
    const int64_t grid = bwd_grid(rows, cols);
    if (workspace_bytes < static_cast<size_t>(grid) * 3 * static_cast<size_t>(cols) * 4)
        return PTXSTD_EINVAL;
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
    p.sums = 1;
    // a single row's gate is a vector gate either way: its gradient is f32 [cols]
    const bool vector_gate = d_gate && gate_rows == 1;
    if (d_w_post) p.post_at = p.sums++;
    if (vector_gate) p.gate_at = p.sums++;
    if (d_gate && !vector_gate) p.dgate_rows = static_cast<uint16_t*>(d_dgate);
    p.gate_stride = vector_gate ? 0 : static_cast<size_t>(cols);
    p.partial = static_cast<float*>(d_workspace);
    auto s = static_cast<cudaStream_t>(stream);
    const uint32_t threads = bwd_threads(cols), g = static_cast<uint32_t>(grid);
    const int v = bwd_vectors(cols);
    int st = v == 1 ? launch_bwd<1>(p, g, threads, s)
             : v == 2 ? launch_bwd<2>(p, g, threads, s) : launch_bwd<4>(p, g, threads, s);
    if (st) return st;
    ptxstd::Reduce r = {};
    r.partial = p.partial;
    r.P = g;
    r.cols = p.sums * p.cols;
    r.split0 = p.cols;
    r.split1 = p.cols * (d_w_post ? 2 : 1);
    r.o0 = d_dw;
    r.o1 = d_dw_post;
    r.o2 = static_cast<float*>(d_dgate);
    return ptxstd::launch_reduce(r, s);
}
