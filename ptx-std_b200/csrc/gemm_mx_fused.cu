// MX GEMMs with an epilogue, on the 5th-generation tensor cores:
//   linear:  pre = A B^T + bias,  result = act(pre) + residual
//   gated:   gate = A Wg^T, up = A Wu^T,  result = act(gate) * up   (one kernel, A read once)
// Operands as for ptxstd_gemm_mx (kind::mxf8f6f4 block32, any pair of element types), results as
// bf16, as an MX operand (E4M3 / E5M2 + blocked UE8M0 scales) for the next GEMM, or both. The f32
// accumulator is biased, activated, multiplied and added to in f32 and rounded once, to bf16 or
// straight to the 8-bit code (no bf16 step between).
//
// Two kernels share that contract:
//
// 1. wide_kernel, for many rows: the CTA-pair pipeline of gemm_mxfp8.cu (256 x 256 tiles of
//    cta_group::2 MMAs, a ring of 128-element K stages, eight epilogue warps per CTA). For the gated
//    product the pair's 256 B rows are 128 rows of Wg (loaded by CTA 0) and the same 128 of Wu (by
//    CTA 1), so the accumulator's columns 0..127 are gate and 128..255 up for the same 128
//    features; an epilogue warp takes 64 columns of each, and the product needs no exchange. A
//    lane holds one row, so the 32 elements of an MX block are in one thread's registers and the
//    block's scale takes no shuffle.
//    Ragged sizes: TMA fills rows and K elements outside the tensors with zeros and clips the
//    stores; MMAs of a last K stage whose 32 elements lie outside are not issued, so padding
//    scales (which may be NaN codes) never meet a product that is kept.
//    Bound by the tensor cores: a stage (256 x 256 x 128) keeps a pair's pipes busy for 512 clocks
//    and takes 602 clocks of the SMs' active time at 4096 x 8192 x 8192, 591 in the gated
//    2048 x 14336 x 4096 (ncu, cold caches; the pipes are active 85 and 87 % of the time). Of the
//    remainder only the pause between two tiles, about 400 clocks or 6 to 13 per stage, is accounted
//    for. The 1 kW power cap sets the clock: 8192^3 takes 361 us (3.05 PFLOP/s, 0.93 of twice the
//    measured bf16 burst) on a cool GPU and 377 to 415 us under load. The epilogue runs beside the
//    next tile's MMAs and shows only when K is short: 4096 x 4096 x 1024 takes 19.1 us plain, 24.8 us
//    with a residual, 31.7 us with bias, GELU and an E4M3 result.
//
// 2. narrow_kernel, for few rows (serving): weight streaming, bound by HBM. The operands swap: 128
//    weight rows are the M side of a cta_group::1 MMA and the tokens (up to 256, a multiple of 16)
//    the N side, so a token costs one accumulator column instead of a padded row. K is split
//    over a cluster; the CTAs' partial accumulators meet in distributed shared memory and are
//    added in rank order, each CTA finishing every S-th token, so the split needs no workspace,
//    no atomics and no second kernel, and the result is reproducible. One token: N = 8192,
//    K = 28672 with residual 38.0 us, 6.4 TB/s or 0.97 of the measured copy rate; gated
//    F = 28672, K = 8192 77.6 us, 0.95 of it. With tens of tokens and mid-sized weights the CTAs'
//    start and end (about 4 us) and an uneven number of blocks per SM cost more: 48 tokens,
//    F = 10240, K = 4096 18.4 us against 13.4 us of HBM time.
//
// Every device-side wait is bounded; a timeout records PTXSTD_ETIMEOUT.
#include <atomic>

#include "common.cuh"
#include "data_types.cuh"
#include "epilogue.cuh"
#include "mx_block.cuh"
#include "tcgen05.cuh"
#include "tma_host.h"

namespace {

namespace t5 = ptxstd::tcgen05;
namespace dt = ptxstd::data_types;
namespace mx = ptxstd::mx;
using ptxstd::mbar_wait;

constexpr uint32_t BK = 128;            // K elements (= bytes) per stage
constexpr uint32_t kMmaK = 32;          // K elements of one mxf8f6f4 MMA
constexpr uint32_t kMmas = BK / kMmaK;  // 4 per stage, one scale byte each
// One step of both scale-factor ids of the instruction descriptor (A's at bits 29-30, B's at bits
// 4-5): MMA j of a stage reads scale byte j.
constexpr uint32_t kScaleIdStep = (1u << 29) | (1u << 4);

// What the epilogues read and write besides the tensor maps.
struct Epi {
    const uint16_t* bias;
    const uint16_t* residual;
    uint16_t* c;     // bf16 result, or null
    uint16_t* pre;   // bf16 pre-activation (linear) / gate projection (gated), or null
    uint16_t* up;    // bf16 up projection (gated), or null
    uint8_t* q;      // MX payload, or null
    uint8_t* sfq;
    uint32_t q_type;
    uint32_t act;
};

__device__ __forceinline__ float f(uint32_t r) { return __uint_as_float(r); }

// ---------------------------------------------------------------------------------------------
// Many rows: CTA pairs, 256-row tiles
// ---------------------------------------------------------------------------------------------
namespace wide {

constexpr uint32_t P_BM = 256, P_BN = 256, P_HALF = 128;
// Five stages, not the six that would fit: the mainloop runs as fast (8192^3 on a cool GPU, with
// raster groups of 8: 372.6 us with five, 372.2 us with six, 389 us with four), and the epilogue
// warps get three staging buffers each: with a residual, 4096 x 4096 x 1024 takes 24.8 us, and took
// 40.6 us with one buffer and the residual read by each lane from its own row.
constexpr uint32_t STAGES = 5;
constexpr uint32_t kEpiWarps = 8;
// Warpgroup 0 holds the producer and MMA warps and needs few registers; the two epilogue
// warpgroups hold 128 accumulator columns per thread and take what it gives up (setmaxnreg). The
// kernel is launched at 168 registers for 384 threads: 128 x 80 + 256 x 208 stay within that.
constexpr uint32_t kFirstEpiWarp = 4;
constexpr uint32_t kThreads = 32 * (kFirstEpiWarp + kEpiWarps);
constexpr uint32_t kRegsCtl = 80, kRegsEpi = 208;
static_assert(128 * kRegsCtl + 256 * kRegsEpi <= 168 * kThreads, "register split");
constexpr uint32_t kABytes = P_HALF * BK;
constexpr uint32_t kBBytes = P_HALF * BK;
constexpr uint32_t kSfaBytes = 512;
constexpr uint32_t kSfbBytes = (P_BN / 128) * 512;
constexpr uint32_t kCtaStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
constexpr uint32_t kSlotCols = 4 + 4 * (P_BN / 128);
constexpr uint32_t kSfBase = P_BN;
constexpr uint32_t kTmemCols = 512;
static_assert(kSfBase + STAGES * kSlotCols <= kTmemCols, "TMEM budget");
constexpr uint32_t kGroupM = 16;  // 8192^3, cool: 361 us, against 372 us with 8 and 381 us with 4
constexpr uint32_t kCCols = 32;   // bf16 columns (or 64 MX bytes) per epilogue store
using StageBox = ptxstd::epi::Box<kCCols>;
constexpr uint32_t kBuffers = 3;  // staging buffers of an epilogue warp

struct alignas(1024) Smem {
    uint8_t a[STAGES][kABytes];
    uint8_t b[STAGES][kBBytes];
    uint8_t sfa[STAGES][kSfaBytes];
    uint8_t sfb[STAGES][kSfbBytes];
    uint8_t cstage[kEpiWarps][kBuffers][StageBox::kBytes];
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t res_full[kEpiWarps][kBuffers];
    uint64_t tfull;
    uint64_t tempty;
    uint64_t drain;
    uint32_t tmem_base;
    uint32_t abort;
};
static_assert(sizeof(Smem::cstage) % 1024 == 0 && (STAGES * (kSfaBytes + kSfbBytes)) % 512 == 0,
              "staging buffers on swizzle boundaries");
constexpr size_t kSmemBytes = sizeof(Smem) + 1024;
static_assert(kSmemBytes <= 232448, "shared memory budget");

enum : uint32_t { kDetailProducer = 0x3500, kDetailMma = 0x3600, kDetailEpilogue = 0x3700 };

struct Maps {
    CUtensorMap a, sfa;
    CUtensorMap b, sfb;    // linear: B; gated: Wg
    CUtensorMap b2, sfb2;  // gated: Wu
    CUtensorMap c, pre, up, q, residual;
};

__device__ __forceinline__ void tile_coords(uint32_t t, uint32_t num_m, uint32_t num_n,
                                            uint32_t& mb, uint32_t& nb) {
    const uint32_t group_tiles = kGroupM * num_n;
    const uint32_t g = t / group_tiles;
    const uint32_t first_m = g * kGroupM;
    const uint32_t gm = min(num_m - first_m, kGroupM);
    const uint32_t local = t - g * group_tiles;
    mb = first_m + local % gm;
    nb = local / gm;
}

__device__ __forceinline__ void fail(Smem& s, uint32_t* err, uint32_t detail) {
    ptxstd::record_error(err, PTXSTD_ETIMEOUT, detail);
    *reinterpret_cast<volatile uint32_t*>(&s.abort) = 1u;
}
__device__ __forceinline__ bool aborted(Smem& s) {
    return *reinterpret_cast<volatile uint32_t*>(&s.abort) != 0u;
}

__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                         uint32_t idesc, uint32_t sfa_tmem, uint32_t sfb_tmem,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate)
        : "memory");
}

// One epilogue warp: its 32 rows of a tile, and its staging buffers. Results leave by TMA stores
// from the buffers in turn, so that a buffer is rewritten when its store of three stores ago has
// been read. A residual comes the other way: boxes of 32 columns are prefetched into the buffers
// before the accumulator is complete, each lane adds its row's values, and the bf16 result is
// written over them and stored from there.
struct EpiWarp {
    uint32_t stg, lane;        // .shared::cta address of buffer 0
    uint64_t* res_full;        // one mbarrier per buffer
    uint32_t next = 0;         // buffer of the next store, without a residual
    uint32_t res_parity = 0;   // bit b: the parity that buffer b's next load completes
    int32_t row0;
    uint32_t row, M, N;        // this lane's row; the result's sizes

    __device__ __forceinline__ uint32_t buffer(uint32_t b) const {
        return stg + b * StageBox::kBytes;
    }
    __device__ __forceinline__ bool live(uint32_t col) const {
        return col < N && static_cast<uint32_t>(row0) < M;
    }
    // The next buffer of the rotation, free to be written.
    __device__ __forceinline__ uint32_t rotate() {
        ptxstd::epi::wait_staging<kBuffers - 1>(lane);
        const uint32_t b = next;
        next = next + 1 == kBuffers ? 0 : next + 1;
        return buffer(b);
    }
    // 32 bf16 columns r[FIRST..] at col through the (free) buffer `at`.
    template <uint32_t FIRST, uint32_t L>
    __device__ __forceinline__ void store_bf16(const CUtensorMap* map, const uint32_t (&r)[L],
                                               uint32_t col, uint32_t at) const {
        ptxstd::epi::stage_store<kCCols, FIRST>(map, at, r, 1.0f, static_cast<int32_t>(col), row0,
                                                lane);
    }
    template <uint32_t FIRST, uint32_t L>
    __device__ __forceinline__ void bf16(const CUtensorMap* map, const uint32_t (&r)[L],
                                         uint32_t col) {
        if (live(col)) store_bf16<FIRST>(map, r, col, rotate());
    }
    // Residual columns col .. + 31 into buffer b (free: nothing still reads it).
    __device__ __forceinline__ void load_residual(const CUtensorMap* map, uint32_t col,
                                                  uint32_t b) const {
        if (lane == 0 && live(col)) {
            ptxstd::mbar_arrive_expect_tx(&res_full[b], StageBox::kBytes);
            asm volatile(
                "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                " [%0], [%1, {%3, %4}], [%2];" ::"r"(buffer(b)),
                "l"(reinterpret_cast<uint64_t>(map)), "r"(ptxstd::smem_u32(&res_full[b])),
                "r"(col), "r"(row0)
                : "memory");
        }
    }
    // Adds buffer b's residual to r[FIRST..]; false after a timeout.
    template <uint32_t FIRST, uint32_t L>
    __device__ __forceinline__ bool add_residual(uint32_t (&r)[L], uint32_t b) {
        const bool ok = mbar_wait(&res_full[b], (res_parity >> b) & 1u);
        res_parity ^= 1u << b;
#pragma unroll
        for (uint32_t c = 0; c < StageBox::kChunks; ++c) {
            uint32_t v[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                         : "r"(buffer(b) + StageBox::offset(lane, c))
                         : "memory");
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                const uint32_t i = FIRST + 8 * c + 2 * k;
                r[i] = __float_as_uint(f(r[i]) + dt::bf16_lo(v[k]));
                r[i + 1] = __float_as_uint(f(r[i + 1]) + dt::bf16_hi(v[k]));
            }
        }
        __syncwarp();  // every lane has read its row
        return ok;
    }
    // Two MX blocks r[FIRST .. FIRST + 63] at col through the (free) buffer `at`; returns their
    // scale codes (0 outside N or M).
    template <uint32_t FIRST, uint32_t L>
    __device__ __forceinline__ uint32_t mx2(const CUtensorMap* map, const uint32_t (&r)[L],
                                            uint32_t col, uint32_t type, uint32_t at) const {
        uint32_t codes = 0;
        const uint32_t emax = mx::emax_of(type);
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            float m = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < 32; i += 2)
                m = mx::amax(m, f(r[FIRST + 32 * h + i]), f(r[FIRST + 32 * h + i + 1]));
            const mx::Scale sc = mx::scale_of(m, emax);
            if (row < M && col + 32 * h < N) codes |= sc.code << (8 * h);
#pragma unroll
            for (uint32_t c = 0; c < 2; ++c) {
                float v[16];
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k) v[k] = f(r[FIRST + 32 * h + 16 * c + k]);
                const uint2 lo = mx::pack8(type, v, sc.inv), hi = mx::pack8(type, v + 8, sc.inv);
                ptxstd::st_shared_v4(at + StageBox::offset(lane, 2 * h + c), lo.x, lo.y, hi.x,
                                     hi.y);
            }
        }
        ptxstd::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            ptxstd::tma_store_2d(map, at, static_cast<int32_t>(col), row0);
            ptxstd::bulk_commit_group();
        }
        return codes;
    }
};

// Adds the bias of columns FIRST .. FIRST + 31 of the warp's 128: lane l holds those of columns
// 4 l .. 4 l + 3.
template <uint32_t FIRST, uint32_t L>
__device__ __forceinline__ void add_bias32(uint32_t (&r)[L], const float (&bias)[4]) {
#pragma unroll
    for (uint32_t i = FIRST; i < FIRST + 32; ++i)
        r[i] = __float_as_uint(f(r[i]) + __shfl_sync(0xffffffffu, bias[i & 3u], (i >> 2) & 31u));
}

template <uint32_t FIRST, uint32_t L>
__device__ __forceinline__ void act32(uint32_t (&r)[L], uint32_t kind) {
    if (kind == PTXSTD_ACT_NONE) return;
    mx::with_act(kind, [&](auto k) {
#pragma unroll
        for (uint32_t i = FIRST; i < FIRST + 32; i += 2) {
            const float2 v =
                ptxstd::unpack2(mx::act2<decltype(k)::value>(ptxstd::pack2f(f(r[i]), f(r[i + 1]))));
            r[i] = __float_as_uint(v.x);
            r[i + 1] = __float_as_uint(v.y);
        }
    });
}

// The buffers that hold residual boxes: all of them while nothing but the bf16 result is stored
// (which replaces the residual in place), else two, the third being the other results'.
__device__ __forceinline__ uint32_t residual_buffers(const Epi& e) {
    return e.pre || e.q ? kBuffers - 1 : kBuffers;
}

// The linear epilogue of 32 accumulator columns r[32 J..], the J-th box of the warp's 128 columns
// from `col0` on. False after a timeout.
template <uint32_t J>
__device__ __forceinline__ bool linear32(uint32_t (&r)[128], EpiWarp& w, const Epi& e,
                                         const Maps& maps, uint32_t col0, const float (&bias)[4]) {
    constexpr uint32_t FIRST = 32 * J;
    const uint32_t col = col0 + FIRST;
    const bool live = w.live(col);
    if (e.bias) add_bias32<FIRST>(r, bias);
    if (e.pre && live) {
        if (e.residual) {
            ptxstd::epi::wait_staging<0>(w.lane);
            w.store_bf16<FIRST>(&maps.pre, r, col, w.buffer(kBuffers - 1));
        } else {
            w.store_bf16<FIRST>(&maps.pre, r, col, w.rotate());
        }
    }
    act32<FIRST>(r, e.act);
    if (!e.residual) {
        if (e.c && live) w.store_bf16<FIRST>(&maps.c, r, col, w.rotate());
        return true;
    }
    bool ok = true;
    const uint32_t n = residual_buffers(e), b = J % n;
    if (live) {
        ok = w.add_residual<FIRST>(r, b);
        if (e.c) w.store_bf16<FIRST>(&maps.c, r, col, w.buffer(b));
    }
    // the next box that has no buffer yet, into the one that is free first
    if (n == kBuffers) {
        if (J == 1) {
            ptxstd::epi::wait_staging<1>(w.lane);  // box 0's store has been read
            w.load_residual(&maps.residual, col0 + 96, 0);
        }
    } else if (J < 2) {
        ptxstd::epi::wait_staging<0>(w.lane);
        w.load_residual(&maps.residual, col + 64, b);
    }
    return ok;
}

// h = act(gate) * up for 32 columns: gate r[FIRST..], up r[64 + FIRST..]; h replaces gate.
template <uint32_t FIRST>
__device__ __forceinline__ void gated32(uint32_t (&r)[128], EpiWarp& w, const Epi& e,
                                        const Maps& maps, uint32_t col) {
    if (e.pre) {
        w.bf16<FIRST>(&maps.pre, r, col);
        w.bf16<64 + FIRST>(&maps.up, r, col);
    }
    act32<FIRST>(r, e.act);
#pragma unroll
    for (uint32_t i = 0; i < 32; ++i)
        r[FIRST + i] = __float_as_uint(f(r[FIRST + i]) * f(r[64 + FIRST + i]));
    if (e.c) w.bf16<FIRST>(&maps.c, r, col);
}

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
    wide_kernel(const __grid_constant__ Maps maps, uint32_t M, uint32_t N, uint32_t K,
                uint32_t atype, uint32_t btype, const __grid_constant__ Epi e, uint32_t* err) {
    constexpr uint32_t kTileN = GATED ? 128 : 256;  // result columns of a tile
    extern __shared__ uint8_t smem_raw[];
    Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                       ~static_cast<uintptr_t>(1023));
    const uint32_t warp = ptxstd::warp_id();
    const uint32_t lane = ptxstd::lane_id();
    const uint32_t rank = ptxstd::cluster_ctarank();
    const uint32_t pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t num_m = (M + P_BM - 1) / P_BM, num_n = (N + kTileN - 1) / kTileN;
    const uint32_t num_tiles = num_m * num_n, num_k = (K + BK - 1) / BK;

    if (warp == 0 && lane == 0) {
        ptxstd::prefetch_tensormap(&maps.a);
        ptxstd::prefetch_tensormap(&maps.b);
        ptxstd::prefetch_tensormap(&maps.sfa);
        ptxstd::prefetch_tensormap(&maps.sfb);
        if (GATED) {
            ptxstd::prefetch_tensormap(&maps.b2);
            ptxstd::prefetch_tensormap(&maps.sfb2);
        }
        for (uint32_t i = 0; i < STAGES; ++i) {
            ptxstd::mbar_init(&s.full[i], 1);
            ptxstd::mbar_init(&s.empty[i], 1);
        }
        ptxstd::mbar_init(&s.tfull, 1);
        ptxstd::mbar_init(&s.tempty, 2 * kEpiWarps);
        ptxstd::mbar_init(&s.drain, 1);
        for (uint32_t i = 0; i < kEpiWarps * kBuffers; ++i)
            ptxstd::mbar_init(&s.res_full[0][0] + i, 1);
        s.abort = 0;
        ptxstd::fence_mbarrier_init();
    }
    if (warp == 1) {
        t5::tmem_alloc_pair(&s.tmem_base, kTmemCols);
        t5::tmem_relinquish_pair();
    }
    t5::fence_before_thread_sync();
    ptxstd::cluster_sync();
    t5::fence_after_thread_sync();
    const uint32_t tmem = s.tmem_base;
    // Only now, with this CTA's TMEM allocated: a dependent CTA on the same SM allocates its own
    // before it waits for this grid, and must not be able to take what this one still needs.
    ptxstd::pdl_launch_dependents();
    ptxstd::pdl_wait();

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        ptxstd::setmaxnreg_dec<kRegsCtl>();
        if (ptxstd::elect_one()) {
            const CUtensorMap* mb_ = GATED && rank == 1 ? &maps.b2 : &maps.b;
            uint32_t stage = 0, phase = 0, issued = 0, issued_parity = 0;
            for (uint32_t t = pair; t < num_tiles && !aborted(s); t += n_pairs) {
                uint32_t mb, nb;
                tile_coords(t, num_m, num_n, mb, nb);
                const int32_t b_row =
                    static_cast<int32_t>(GATED ? nb * 128 : nb * P_BN + rank * P_HALF);
                for (uint32_t kb = 0; kb < num_k; ++kb) {
                    if (!mbar_wait(&s.empty[stage], phase ^ 1u)) {
                        fail(s, err, kDetailProducer | stage);
                        break;
                    }
                    if (aborted(s)) break;
                    const uint32_t fl = ptxstd::mapa_shared(ptxstd::smem_u32(&s.full[stage]), 0);
                    if (rank == 0) ptxstd::mbar_arrive_expect_tx(&s.full[stage], 2 * kCtaStageBytes);
                    ptxstd::tma_load_2d_pair(s.a[stage], &maps.a, fl, static_cast<int32_t>(kb * BK),
                                             static_cast<int32_t>(mb * P_BM + rank * P_HALF));
                    ptxstd::tma_load_2d_pair(s.b[stage], mb_, fl, static_cast<int32_t>(kb * BK),
                                             b_row);
                    ptxstd::tma_load_2d_pair(s.sfa[stage], &maps.sfa, fl, 0,
                                             static_cast<int32_t>((mb * 2 + rank) * num_k + kb));
                    if constexpr (GATED) {
                        ptxstd::tma_load_2d_pair(s.sfb[stage], &maps.sfb, fl, 0,
                                                 static_cast<int32_t>(nb * num_k + kb));
                        ptxstd::tma_load_2d_pair(s.sfb[stage] + 512, &maps.sfb2, fl, 0,
                                                 static_cast<int32_t>(nb * num_k + kb));
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < P_BN / 128; ++j)
                            ptxstd::tma_load_2d_pair(
                                s.sfb[stage] + j * 512, &maps.sfb, fl, 0,
                                static_cast<int32_t>((nb * 2 + j) * num_k + kb));
                    }
                    issued |= 1u << stage;
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (aborted(s) && rank == 0) {
                for (uint32_t i = 0; i < STAGES; ++i)
                    if (issued & (1u << i)) mbar_wait(&s.full[i], (issued_parity >> i) & 1u);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader) ----------------
        ptxstd::setmaxnreg_dec<kRegsCtl>();
        // The whole warp runs the loops and one lane issues: with uniform control flow the operands
        // stay in uniform registers, which the tensor instructions take them from. (Inside a loop
        // of one elected lane the compiler did that for some epilogues and not for others, and
        // then a stage took 888 clocks to issue instead of 430: 8192^3 in 443 us, not 361 us.)
        if (rank == 0) {
            const bool lead = ptxstd::elect_one();
            uint32_t idesc = 0;
            t5::idesc_mxf8f6f4(atype, btype, P_BM, P_BN, idesc);
            const uint64_t a0 = t5::smem_desc_k128(ptxstd::smem_u32(s.a[0]));
            const uint64_t b0 = t5::smem_desc_k128(ptxstd::smem_u32(s.b[0]));
            const uint64_t sfa0 = t5::smem_desc_nosw(ptxstd::smem_u32(s.sfa[0]), 0, 128);
            const uint64_t sfb0 = t5::smem_desc_nosw(ptxstd::smem_u32(s.sfb[0]), 0, 128);
            const uint32_t empty0 = ptxstd::smem_u32(&s.empty[0]);
            const uint32_t peer_empty0 = ptxstd::mapa_shared(empty0, 1);
            const uint32_t tfull = ptxstd::smem_u32(&s.tfull);
            const uint32_t peer_tfull = ptxstd::mapa_shared(tfull, 1);
            uint32_t stage = 0, phase = 0, acc_phase = 0;
            for (uint32_t t = pair; t < num_tiles; t += n_pairs) {
                if (!__all_sync(0xffffffffu, !aborted(s) && mbar_wait(&s.tempty, acc_phase ^ 1u))) {
                    if (lead && !aborted(s)) fail(s, err, kDetailMma | 0x90);
                    break;
                }
                t5::fence_after_thread_sync();
                bool ok = true;
                for (uint32_t kb = 0; kb < num_k; ++kb) {
                    if (!__all_sync(0xffffffffu, mbar_wait(&s.full[stage], phase))) {
                        if (lead) fail(s, err, kDetailMma | 0x80 | stage);
                        ok = false;
                        break;
                    }
                    t5::fence_after_thread_sync();
                    const uint64_t ad = a0 + stage * (kABytes >> 4);
                    const uint64_t bd = b0 + stage * (kBBytes >> 4);
                    const uint64_t sfa = sfa0 + stage * (kSfaBytes >> 4);
                    const uint64_t sfb = sfb0 + stage * (kSfbBytes >> 4);
                    const uint32_t slot = tmem + kSfBase + stage * kSlotCols;
                    const uint32_t live = (K - kb * BK) / kMmaK;  // MMAs inside K
                    if (lead) {
                        t5::cp_32x128b_warpx4_pair(slot, sfa);
#pragma unroll
                        for (uint32_t h = 0; h < P_BN / 128; ++h)
                            t5::cp_32x128b_warpx4_pair(slot + 4 + 4 * h, sfb + 32 * h);
#pragma unroll
                        for (uint32_t j = 0; j < kMmas; ++j)
                            if (j < live)
                                mma_pair(tmem, ad + 2 * j, bd + 2 * j, idesc + j * kScaleIdStep,
                                         slot, slot + 4, (kb | j) != 0u);
                        t5::commit_pair(empty0 + 8 * stage);
                        t5::commit_pair(peer_empty0 + 8 * stage);
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (lead) {
                    t5::commit_pair(tfull);
                    t5::commit_pair(peer_tfull);
                }
                acc_phase ^= 1u;
            }
            if (lead) {
                t5::commit_pair(ptxstd::smem_u32(&s.drain));
                mbar_wait(&s.drain, 0);
            }
            __syncwarp();
        }
    } else if (warp < kFirstEpiWarp) {
        ptxstd::setmaxnreg_dec<kRegsCtl>();  // idle: its share of registers goes to the epilogue
    } else {
        // ---------------- epilogue: warps 4..11 of both CTAs ----------------
        ptxstd::setmaxnreg_inc<kRegsEpi>();
        const uint32_t ew = warp - kFirstEpiWarp, q = warp & 3u, half = ew >> 2;
        uint32_t acc_phase = 0;
        const uint32_t tempty_leader = ptxstd::mapa_shared(ptxstd::smem_u32(&s.tempty), 0);
        const size_t q_tiles_k = mx::tiles_k(N / 32);
        EpiWarp w;
        w.stg = ptxstd::smem_u32(s.cstage[ew][0]);
        w.lane = lane;
        w.res_full = s.res_full[ew];
        w.M = M;
        w.N = N;
        for (uint32_t t = pair; t < num_tiles; t += n_pairs) {
            uint32_t mb, nb;
            tile_coords(t, num_m, num_n, mb, nb);
            w.row0 = static_cast<int32_t>(mb * P_BM + rank * P_HALF + 32 * q);
            w.row = static_cast<uint32_t>(w.row0) + lane;
            const uint32_t col0 = nb * kTileN + half * (GATED ? 64 : 128);
            // while the accumulator is being computed: the bias to registers, residual boxes to the
            // staging buffers (the bias by an ordinary load: under programmatic launch the kernel before
            // may write it while this grid is resident, which ld.global.nc does not allow for)
            float bias[4] = {};
            if (!GATED && e.bias && col0 + 4 * lane < N) {
                const uint2 v = *reinterpret_cast<const uint2*>(e.bias + col0 + 4 * lane);
                bias[0] = dt::bf16_lo(v.x);
                bias[1] = dt::bf16_hi(v.x);
                bias[2] = dt::bf16_lo(v.y);
                bias[3] = dt::bf16_hi(v.y);
            }
            if (!GATED && e.residual) {
                ptxstd::epi::wait_staging<0>(lane);
                const uint32_t n = residual_buffers(e);
                for (uint32_t b = 0; b < n; ++b) w.load_residual(&maps.residual, col0 + 32 * b, b);
            }

            bool ok = !aborted(s) && mbar_wait(&s.tfull, acc_phase);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0 && !aborted(s)) fail(s, err, kDetailEpilogue | 0x80);
                // the residual boxes under way have to land before this block may end
                if (!GATED && e.residual)
                    for (uint32_t b = 0; b < residual_buffers(e); ++b)
                        if (w.live(col0 + 32 * b))
                            mbar_wait(&w.res_full[b], (w.res_parity >> b) & 1u);
                break;
            }
            t5::fence_after_thread_sync();
            // linear: accumulator columns 128 half .. + 127; gated: gate columns 64 half .. + 63,
            // then up columns 128 + 64 half .. + 63
            uint32_t r[128];
            const uint32_t lo = tmem + ((32 * q) << 16) + half * (GATED ? 64 : 128);
            const uint32_t hi = lo + (GATED ? 128 : 64);
            {
                uint32_t(&r0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&r[0]);
                uint32_t(&r1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&r[32]);
                uint32_t(&r2)[32] = *reinterpret_cast<uint32_t(*)[32]>(&r[64]);
                uint32_t(&r3)[32] = *reinterpret_cast<uint32_t(*)[32]>(&r[96]);
                t5::ld_32x32b_x32(lo, r0);
                t5::ld_32x32b_x32(lo + 32, r1);
                t5::ld_32x32b_x32(hi, r2);
                t5::ld_32x32b_x32(hi + 32, r3);
                t5::wait_ld();
            }
            t5::fence_before_thread_sync();
            __syncwarp();
            if (lane == 0) ptxstd::mbar_arrive_cluster_relaxed(tempty_leader);
            acc_phase ^= 1u;

            const bool in_tiles = w.row < mx::padded_rows(M);  // a row of the scale tiles
            if constexpr (GATED) {
                gated32<0>(r, w, e, maps, col0);
                gated32<32>(r, w, e, maps, col0 + 32);
                if (e.q) {
                    uint32_t codes = 0;
                    if (w.live(col0)) codes = w.mx2<0>(&maps.q, r, col0, e.q_type, w.rotate());
                    // the tile's four scale columns: this warp holds two of them
                    if (in_tiles)
                        *reinterpret_cast<uint16_t*>(
                            e.sfq + mx::word_offset(w.row, nb, q_tiles_k) + 2 * half) =
                            static_cast<uint16_t>(codes);
                }
            } else {
                // with a residual the MX results take the last buffer, else the rotation's
                auto mx_buffer = [&] {
                    if (!e.residual) return w.rotate();
                    ptxstd::epi::wait_staging<0>(lane);
                    return w.buffer(kBuffers - 1);
                };
                uint32_t codes = 0;
                ok = linear32<0>(r, w, e, maps, col0, bias);
                ok &= linear32<1>(r, w, e, maps, col0, bias);
                if (e.q && w.live(col0)) codes = w.mx2<0>(&maps.q, r, col0, e.q_type, mx_buffer());
                ok &= linear32<2>(r, w, e, maps, col0, bias);
                ok &= linear32<3>(r, w, e, maps, col0, bias);
                if (e.q && w.live(col0 + 64))
                    codes |= w.mx2<64>(&maps.q, r, col0 + 64, e.q_type, mx_buffer()) << 16;
                if (e.q && in_tiles && col0 < N)
                    *reinterpret_cast<uint32_t*>(
                        e.sfq + mx::word_offset(w.row, nb * 2 + half, q_tiles_k)) = codes;
                // a residual that did not arrive: recorded, and the other roles stop
                if (__any_sync(0xffffffffu, !ok) && lane == 0)
                    fail(s, err, kDetailEpilogue | 0x40);
            }
        }
        ptxstd::epi::drain(lane);
    }

    t5::fence_before_thread_sync();
    ptxstd::cluster_sync();
    t5::fence_after_thread_sync();
    if (warp == 1) t5::tmem_dealloc_pair(tmem, kTmemCols);
}

}  // namespace wide

// ---------------------------------------------------------------------------------------------
// Few rows: weights on the M side, tokens on the N side, K split over a cluster
// ---------------------------------------------------------------------------------------------
namespace narrow {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWBytes = 128 * BK;  // one weight tile of a stage
constexpr uint32_t kMaxStages = 12;

enum : uint32_t { kDetailProducer = 0x3900, kDetailMma = 0x3A00, kDetailEpilogue = 0x3B00 };

struct Maps {
    CUtensorMap x, sfx;
    CUtensorMap w, sfw;    // linear: B; gated: Wg
    CUtensorMap w2, sfw2;  // gated: Wu
};

struct Shape {
    uint32_t M, N, K;
    uint32_t tokens;    // token columns of a CTA: a multiple of 16, up to 256
    uint32_t stages;
    uint32_t split;     // CTAs of a cluster = K slices
    uint32_t tmem_cols;
};

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

struct Bars {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t done;
    uint32_t tmem_base;
    uint32_t abort;
};

__device__ __forceinline__ void act8(float (&v)[8], uint32_t kind) {
    if (kind == PTXSTD_ACT_NONE) return;
    mx::with_act(kind, [&](auto k) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i += 2) {
            const float2 y =
                ptxstd::unpack2(mx::act2<decltype(k)::value>(ptxstd::pack2f(v[i], v[i + 1])));
            v[i] = y.x;
            v[i + 1] = y.y;
        }
    });
}

// The sum of a row chunk's partials over the cluster's CTAs, in rank order: eight columns at byte
// `at` of every CTA's partial buffer. All loads are issued before the first add.
template <uint32_t S>
__device__ __forceinline__ void sum_peers(const uint32_t (&peer)[S], uint32_t at, float (&v)[8]) {
    float4 lo[S], hi[S];
#pragma unroll
    for (uint32_t s = 0; s < S; ++s) {
        lo[s] = ld_cluster_v4(peer[s] + at);
        hi[s] = ld_cluster_v4(peer[s] + at + 16);
    }
    v[0] = lo[0].x, v[1] = lo[0].y, v[2] = lo[0].z, v[3] = lo[0].w;
    v[4] = hi[0].x, v[5] = hi[0].y, v[6] = hi[0].z, v[7] = hi[0].w;
#pragma unroll
    for (uint32_t s = 1; s < S; ++s) {
        v[0] += lo[s].x, v[1] += lo[s].y, v[2] += lo[s].z, v[3] += lo[s].w;
        v[4] += hi[s].x, v[5] += hi[s].y, v[6] += hi[s].z, v[7] += hi[s].w;
    }
}

// The epilogue proper: 16 threads per token, eight result columns (weight rows) each; CTA `rank`
// takes the tokens rank, rank + S, ... of the tile. With an MX result the padding rows of the last
// scale tile get zero codes.
template <bool GATED, uint32_t S>
__device__ __forceinline__ void narrow_epilogue(const Shape& p, const Epi& e, uint32_t part_addr,
                                                uint32_t rank, uint32_t block, uint32_t tok0,
                                                const float (&bias)[8]) {
    constexpr uint32_t G = GATED ? 2 : 1;
    const uint32_t tid = threadIdx.x, lane = ptxstd::lane_id();
    const uint32_t c8 = (tid & 15u) * 8, col = block * 128 + c8, T = p.tokens;
    const uint32_t live = min(T, p.M - tok0);
    const bool last_y = blockIdx.y + 1 == gridDim.y;
    const uint32_t upto =
        e.q ? (last_y ? static_cast<uint32_t>(mx::padded_rows(p.M)) - tok0 : T) : live;
    const bool col_ok = col < p.N;
    const size_t q_tiles_k = mx::tiles_k(p.N / 32);
    uint32_t peer[S];
#pragma unroll
    for (uint32_t s = 0; s < S; ++s) peer[s] = S > 1 ? ptxstd::mapa_shared(part_addr, s) : part_addr;
    // uniform trip count per warp (the shuffles below take all lanes)
    for (uint32_t t0 = rank; t0 < upto; t0 += 16 * S) {
        const uint32_t t = t0 + (tid >> 4) * S;
        const bool on = t < live && col_ok;
        const size_t at = static_cast<size_t>(tok0 + t) * p.N + col;
        float v[G][8];
        uint4 res = make_uint4(0, 0, 0, 0);
        if (on) {
            if (!GATED && e.residual) res = *reinterpret_cast<const uint4*>(e.residual + at);
#pragma unroll
            for (uint32_t g = 0; g < G; ++g)
                sum_peers<S>(peer, ((g * T + t) * 128 + c8) * 4, v[g]);
        } else {
#pragma unroll
            for (uint32_t g = 0; g < G; ++g)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) v[g][i] = 0.0f;
        }
        auto store_bf16 = [&](uint16_t* dst, const float* x) {
            uint4 o;
            o.x = dt::bf16x2_from_f32(x[0], x[1]);
            o.y = dt::bf16x2_from_f32(x[2], x[3]);
            o.z = dt::bf16x2_from_f32(x[4], x[5]);
            o.w = dt::bf16x2_from_f32(x[6], x[7]);
            *reinterpret_cast<uint4*>(dst + at) = o;
        };
        float y[8];
        if constexpr (GATED) {
            if (on && e.pre) {
                store_bf16(e.pre, v[0]);
                store_bf16(e.up, v[1]);
            }
            act8(v[0], e.act);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) y[i] = v[0][i] * v[G - 1][i];
        } else {
            const uint32_t rw[4] = {res.x, res.y, res.z, res.w};
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) v[0][i] += bias[i];
            if (on && e.pre) store_bf16(e.pre, v[0]);
            act8(v[0], e.act);
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                y[i] = v[0][i] + ((i & 1) ? dt::bf16_hi(rw[i >> 1]) : dt::bf16_lo(rw[i >> 1]));
        }
        if (on && e.c) store_bf16(e.c, y);
        if (e.q) {
            const mx::Scale sc =
                mx::scale_of(mx::amax_quad(mx::amax_of(y)), mx::emax_of(e.q_type));
            if (on) *reinterpret_cast<uint2*>(e.q + at) = mx::pack8(e.q_type, y, sc.inv);
            if ((lane & 3u) == 0 && t < upto)
                e.sfq[mx::word_offset(tok0 + t, block, q_tiles_k) + ((tid & 15u) >> 2)] =
                    on ? static_cast<uint8_t>(sc.code) : 0;
        }
    }
}

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 2)
    narrow_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Shape p,
                  uint32_t wtype, uint32_t xtype, const __grid_constant__ Epi e, uint32_t* err) {
    constexpr uint32_t G = GATED ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars b;
    const uint32_t raw = ptxstd::smem_u32(smem_raw);
    uint8_t* const base = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
    const uint32_t T = p.tokens, tok_tiles = (T + 127) / 128;
    const uint32_t stage_bytes = G * kWBytes + T * BK;
    const uint32_t sf_bytes = (G + tok_tiles) * 512;
    uint8_t* const sf_base = base + p.stages * stage_bytes;
    float* const part = reinterpret_cast<float*>(base);  // after the products: [G][T][128]

    const uint32_t warp = ptxstd::warp_id(), lane = ptxstd::lane_id(), tid = threadIdx.x;
    const uint32_t rank = p.split > 1 ? ptxstd::cluster_ctarank() : 0;
    const uint32_t block = blockIdx.x / p.split;  // 128 weight rows
    const uint32_t num_k = (p.K + BK - 1) / BK;
    const uint32_t k_lo = static_cast<uint32_t>(static_cast<uint64_t>(num_k) * rank / p.split);
    const uint32_t k_hi = static_cast<uint32_t>(static_cast<uint64_t>(num_k) * (rank + 1) / p.split);
    const uint32_t tok0 = blockIdx.y * T;
    volatile uint32_t* abort_flag = &b.abort;

    if (tid == 0) {
        ptxstd::prefetch_tensormap(&maps.x);
        ptxstd::prefetch_tensormap(&maps.w);
        ptxstd::prefetch_tensormap(&maps.sfx);
        ptxstd::prefetch_tensormap(&maps.sfw);
        for (uint32_t i = 0; i < p.stages; ++i) {
            ptxstd::mbar_init(&b.full[i], 1);
            ptxstd::mbar_init(&b.empty[i], 1);
        }
        ptxstd::mbar_init(&b.done, 1);
        b.abort = 0;
        ptxstd::fence_mbarrier_init();
    }
    if (warp == 1) {
        t5::tmem_alloc(&b.tmem_base, p.tmem_cols);
        t5::tmem_relinquish();
    }
    t5::fence_before_thread_sync();
    __syncthreads();
    t5::fence_after_thread_sync();
    const uint32_t tmem = b.tmem_base;
    ptxstd::pdl_launch_dependents();  // after the TMEM allocation, as in the wide kernel
    ptxstd::pdl_wait();
    float bias[8] = {};
    if (!GATED && e.bias && block * 128 + (tid & 15u) * 8 < p.N) {
        const uint4 w = *reinterpret_cast<const uint4*>(e.bias + block * 128 + (tid & 15u) * 8);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            bias[2 * k] = dt::bf16_lo(v[k]);
            bias[2 * k + 1] = dt::bf16_hi(v[k]);
        }
    }

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (ptxstd::elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0, issued_parity = 0;
            for (uint32_t kb = k_lo; kb < k_hi; ++kb) {
                if (!mbar_wait(&b.empty[stage], phase ^ 1u)) {
                    ptxstd::record_error(err, PTXSTD_ETIMEOUT, kDetailProducer | stage);
                    *abort_flag = 1u;
                }
                if (*abort_flag) break;
                uint8_t* const st = base + stage * stage_bytes;
                uint8_t* const sf = sf_base + stage * sf_bytes;
                const int32_t k = static_cast<int32_t>(kb * BK);
                ptxstd::mbar_arrive_expect_tx(&b.full[stage], stage_bytes + sf_bytes);
                ptxstd::tma_load_2d(st, &maps.w, &b.full[stage], k,
                                    static_cast<int32_t>(block * 128));
                if constexpr (GATED)
                    ptxstd::tma_load_2d(st + kWBytes, &maps.w2, &b.full[stage], k,
                                        static_cast<int32_t>(block * 128));
                ptxstd::tma_load_2d(st + G * kWBytes, &maps.x, &b.full[stage], k,
                                    static_cast<int32_t>(tok0));
                ptxstd::tma_load_2d(sf, &maps.sfw, &b.full[stage], 0,
                                    static_cast<int32_t>(block * num_k + kb));
                if constexpr (GATED)
                    ptxstd::tma_load_2d(sf + 512, &maps.sfw2, &b.full[stage], 0,
                                        static_cast<int32_t>(block * num_k + kb));
                for (uint32_t j = 0; j < tok_tiles; ++j)
                    ptxstd::tma_load_2d(sf + (G + j) * 512, &maps.sfx, &b.full[stage], 0,
                                        static_cast<int32_t>((tok0 / 128 + j) * num_k + kb));
                issued |= 1u << stage;
                issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                if (++stage == p.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (*abort_flag) {
                for (uint32_t i = 0; i < p.stages; ++i)
                    if (issued & (1u << i)) mbar_wait(&b.full[i], (issued_parity >> i) & 1u);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (uniform control flow, one lane issues) ----------------
        const bool lead = ptxstd::elect_one();
        uint32_t idesc = 0;
        t5::idesc_mxf8f6f4(wtype, xtype, 128, T, idesc);
        const uint32_t slot_cols = 4 * (G + tok_tiles);
        // a column of the copied scales holds 32 rows: a 64-token tile may start at the third
        const uint32_t x_col = 4 * G + (tok0 % 128) / 32;
        const uint32_t st0 = ptxstd::smem_u32(base), sf0 = ptxstd::smem_u32(sf_base);
        uint32_t stage = 0, phase = 0;
        for (uint32_t kb = k_lo; kb < k_hi; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(&b.full[stage], phase))) {
                if (lead) {
                    ptxstd::record_error(err, PTXSTD_ETIMEOUT, kDetailMma | stage);
                    *abort_flag = 1u;
                }
                break;
            }
            t5::fence_after_thread_sync();
            const uint32_t slot = tmem + G * T + stage * slot_cols;
            const uint64_t sfd = t5::smem_desc_nosw(sf0 + stage * sf_bytes, 0, 128);
            const uint64_t wd = t5::smem_desc_k128(st0 + stage * stage_bytes);
            const uint64_t xd = wd + G * (kWBytes >> 4);
            const uint32_t live = (p.K - kb * BK) / kMmaK;
            if (lead) {
                for (uint32_t j = 0; j < G + tok_tiles; ++j)
                    t5::cp_32x128b_warpx4(slot + 4 * j, sfd + 32 * j);
#pragma unroll
                for (uint32_t g = 0; g < G; ++g)
#pragma unroll
                    for (uint32_t j = 0; j < kMmas; ++j)
                        if (j < live)
                            t5::mma_mxf8f6f4_block32(
                                tmem + g * T, wd + g * (kWBytes >> 4) + 2 * j, xd + 2 * j,
                                idesc + j * kScaleIdStep, slot + 4 * g, slot + x_col,
                                kb > k_lo || j > 0);
                t5::commit(&b.empty[stage]);
            }
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (lead) t5::commit(&b.done);
    }
    __syncwarp();

    // ---------------- every warp: accumulators to shared memory, then the epilogue -----------
    // `done` completes after the last MMA; by then every load has landed, so the ring's memory
    // is free for the partial sums.
    bool ok = mbar_wait(&b.done, 0);
    if (!ok && lane == 0) ptxstd::record_error(err, PTXSTD_ETIMEOUT, kDetailEpilogue);
    ok = __syncthreads_and(ok && !*abort_flag);
    t5::fence_after_thread_sync();
    if (ok) {
        // warp w: lanes 32 (w % 4) .. + 31 of every other 16 columns, two loads in flight
        const uint32_t q = warp & 3u, cols = G * T;
        float* const dst = part + 32 * q + lane;
        for (uint32_t c = (warp >> 2) * 16; c < cols; c += 64) {
            const uint32_t ta = tmem + ((32 * q) << 16) + c;
            const bool two = c + 32 < cols;
            uint32_t r[16], r2[16];
            t5::ld_32x32b_x16(ta, r);
            if (two) t5::ld_32x32b_x16(ta + 32, r2);
            t5::wait_ld();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) dst[(c + i) * 128] = f(r[i]);
            if (two) {
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) dst[(c + 32 + i) * 128] = f(r2[i]);
            }
        }
    }
    t5::fence_before_thread_sync();
    if (p.split > 1) ptxstd::cluster_sync();
    else __syncthreads();
    t5::fence_after_thread_sync();
    if (warp == 1) t5::tmem_dealloc(tmem, p.tmem_cols);

    if (ok) {
        const uint32_t pa = ptxstd::smem_u32(part);
        switch (p.split) {
        case 1: narrow_epilogue<GATED, 1>(p, e, pa, rank, block, tok0, bias); break;
        case 2: narrow_epilogue<GATED, 2>(p, e, pa, rank, block, tok0, bias); break;
        case 3: narrow_epilogue<GATED, 3>(p, e, pa, rank, block, tok0, bias); break;
        case 4: narrow_epilogue<GATED, 4>(p, e, pa, rank, block, tok0, bias); break;
        case 5: narrow_epilogue<GATED, 5>(p, e, pa, rank, block, tok0, bias); break;
        case 6: narrow_epilogue<GATED, 6>(p, e, pa, rank, block, tok0, bias); break;
        default: narrow_epilogue<GATED, 8>(p, e, pa, rank, block, tok0, bias); break;
        }
    }
    // no CTA of the cluster leaves while another may still read its partial sums
    if (p.split > 1) ptxstd::cluster_sync();
}

}  // namespace narrow

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
bool mx_type_ok(int t) { return t == 0 || t == 1 || t == 3 || t == 4 || t == 5; }

struct Operand {
    const uint8_t* data;
    const uint8_t* sf;
};

int operand_maps(CUtensorMap* data, CUtensorMap* sf, Operand o, int64_t rows, int64_t K,
                 uint32_t box_rows) {
    const int st = ptxstd::make_tmap_2d(data, o.data, CU_TENSOR_MAP_DATA_TYPE_UINT8, K, rows, K, BK,
                                        box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
    return ptxstd::make_tmap_2d(sf, o.sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 128,
                                ((rows + 127) / 128) * ((K + 127) / 128), 512, 128, 1,
                                CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <bool GATED>
int launch_wide(Operand a, int a_type, Operand b, Operand b2, int b_type, const Epi& e, int64_t M,
                int64_t N, int64_t K, cudaStream_t stream) {
    using namespace wide;
    Maps maps = {};
    int st = operand_maps(&maps.a, &maps.sfa, a, M, K, P_HALF);
    if (st) return st;
    st = operand_maps(&maps.b, &maps.sfb, b, N, K, P_HALF);
    if (st) return st;
    if (GATED) {
        st = operand_maps(&maps.b2, &maps.sfb2, b2, N, K, P_HALF);
        if (st) return st;
    }
    if (e.c && (st = ptxstd::epi::make_store_map<kCCols>(&maps.c, e.c, M, N))) return st;
    if (e.pre && (st = ptxstd::epi::make_store_map<kCCols>(&maps.pre, e.pre, M, N))) return st;
    if (e.up && (st = ptxstd::epi::make_store_map<kCCols>(&maps.up, e.up, M, N))) return st;
    if (e.residual &&
        (st = ptxstd::epi::make_store_map<kCCols>(&maps.residual,
                                                  const_cast<uint16_t*>(e.residual), M, N)))
        return st;
    if (e.q && (st = ptxstd::make_tmap_2d(&maps.q, e.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, N, M, N, 64,
                                          ptxstd::epi::kRows, CU_TENSOR_MAP_SWIZZLE_64B)))
        return st;
    st = ptxstd::set_max_dynamic_smem(reinterpret_cast<const void*>(wide_kernel<GATED>),
                                      static_cast<int>(kSmemBytes));
    if (st) return st;
    uint32_t* err = ptxstd::device_error_word();
    if (!err) return PTXSTD_ECUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    static std::atomic<int> max_pairs[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return PTXSTD_ECUDA;
    int resident = max_pairs[dev].load(std::memory_order_relaxed);
    if (resident == 0) {
        cfg.gridDim = dim3(2 * static_cast<uint32_t>(ptxstd::sm_count() / 2));
        if (cudaOccupancyMaxActiveClusters(&resident, wide_kernel<GATED>, &cfg) != cudaSuccess ||
            resident <= 0)
            return PTXSTD_ECUDA;
        max_pairs[dev].store(resident, std::memory_order_relaxed);
    }
    cfg.numAttrs = 2;
    const int64_t tile_n = GATED ? 128 : 256;
    const int64_t tiles = ((M + P_BM - 1) / P_BM) * ((N + tile_n - 1) / tile_n);
    if (tiles >= (1ll << 31)) return PTXSTD_EINVAL;
    cfg.gridDim = dim3(2 * static_cast<uint32_t>(tiles < resident ? tiles : resident));
    if (cudaLaunchKernelEx(&cfg, wide_kernel<GATED>, maps, static_cast<uint32_t>(M),
                           static_cast<uint32_t>(N), static_cast<uint32_t>(K),
                           static_cast<uint32_t>(a_type), static_cast<uint32_t>(b_type), e,
                           err) != cudaSuccess)
        return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

// How a narrow call runs: token columns of a CTA, K slices of a cluster, CTAs per SM.
struct NarrowPlan {
    uint32_t tokens, split, stages, tmem_cols, smem;
    double us;  // estimated time
};

constexpr uint32_t kHalfSmem = 111 * 1024, kFullSmem = 225 * 1024;

// The ring of one CTA, with `two` CTAs on an SM or one; false where it does not fit.
bool narrow_ring(NarrowPlan& p, uint32_t G, uint32_t tokens, bool two) {
    using namespace narrow;
    const uint32_t tok_tiles = (tokens + 127) / 128, slot_cols = 4 * (G + tok_tiles);
    const uint32_t per_stage = G * kWBytes + tokens * BK + (G + tok_tiles) * 512;
    p.tokens = tokens;
    p.stages = (two ? kHalfSmem : kFullSmem) / per_stage;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    if (p.stages < 2) return false;
    const uint32_t cols = G * tokens + p.stages * slot_cols;
    if (cols > (two ? 256u : 512u)) return false;
    // TMEM waits inside clusters must not be able to form a cycle, whatever else runs on the GPU
    // (another stream's call, the next call's early start): a CTA that is to be alone takes all of
    // its SM's shared memory and may then have all of its TMEM; the others take half of TMEM and
    // more than a third of the shared memory, so that two is the most an SM holds.
    p.tmem_cols = two ? 256 : 512;
    p.smem = two ? p.stages * per_stage + 1024 : kFullSmem + 1024;
    if (p.smem < 78 * 1024) p.smem = 78 * 1024;
    const uint32_t part = G * tokens * 128 * 4 + 1024;
    return p.smem >= part;
}

// CTAs of a narrow launch that the GPU holds at once with one per SM, in clusters of `split`: asked
// of the runtime once per device and kind (clusters of more than two leave SMs of their processing
// clusters unused, how many depends on the part). 0 where a cluster does not fit.
template <bool GATED>
int64_t narrow_slots(uint32_t split) {
    static std::atomic<int> cache[64][9];  // value + 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    std::atomic<int>& c = cache[dev][split];
    int n = c.load(std::memory_order_relaxed);
    if (n == 0) {
        const void* kernel = reinterpret_cast<const void*>(narrow::narrow_kernel<GATED>);
        if (ptxstd::set_max_dynamic_smem(kernel, kFullSmem + 1024) != PTXSTD_OK) return 0;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = split;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(split);
        cfg.blockDim = dim3(narrow::kThreads);
        cfg.dynamicSmemBytes = kFullSmem + 1024;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        n = clusters * static_cast<int>(split) + 1;
        c.store(n, std::memory_order_relaxed);
    }
    return n - 1;
}

// The plan with the least estimated time, in us. The model was fitted to sweeps of tokens, split
// and CTAs per SM over 1 <= M <= 1000 on a B200 and is mostly within 15 % of the times there (5 to
// 40 us): a launch 2.5; a CTA's start and end 1.5, which CTAs sharing an SM overlap; an SM takes
// in its ring's bytes every 2.1 us, at most 95 GB/s; the partial sums' exchange 1.0 and 30 GB/s,
// half as much again with two accumulators; and all of it no faster than HBM delivers. At M = 200,
// N = 4128, K = 2080 it takes 64-token tiles without a split: 8.0 us, against 10.5 us for one
// 208-token tile split in two and 9.8 us for the wide kernel (all for a plain bf16 result; with bias,
// GELU and an E4M3 result the first takes 9.6 us).
template <bool GATED>
NarrowPlan narrow_plan(int64_t M, int64_t N, int64_t K) {
    const uint32_t G = GATED ? 2 : 1, cap = GATED ? 128 : 256;
    const int64_t blocks = (N + 127) / 128, num_k = (K + BK - 1) / BK;
    const double hbm = 2.5 + static_cast<double>(G) * N * K * (33.0 / 32.0) / 6.4e6;
    NarrowPlan best = {};
    best.us = 1e30;
    const int64_t whole = (M + 15) / 16 * 16;
    // one tile of all tokens, or tiles of 64, 128 or 256 (a tile must not straddle a scale tile)
    for (const int64_t t : {whole, int64_t{64}, int64_t{128}, int64_t{256}}) {
        if (t > cap || (t != whole && t >= M)) continue;
        const int64_t ytiles = (M + t - 1) / t;
        for (const bool two : {false, true}) {
            NarrowPlan p = {};
            if (!narrow_ring(p, G, static_cast<uint32_t>(t), two)) continue;
            const double stage = G * 16896.0 + t * 132.0;
            for (const uint32_t s : {1u, 2u, 3u, 4u, 5u, 6u, 8u}) {
                if (s > 1 && num_k < 2 * s) break;
                const int64_t ctas = blocks * ytiles * s;
                const int64_t slots = narrow_slots<GATED>(s) * (two ? 2 : 1);
                if (slots == 0) continue;
                const int64_t waves = (ctas + slots - 1) / slots;
                // CTAs that share an SM share its intake
                const bool shared = two && ctas > slots / 2;
                const double in_flight = (shared ? 2.0 : 1.0) * (p.stages - 0.5) * stage;
                const double rate = in_flight / 2.1 < 95e3 ? in_flight / 2.1 : 95e3;
                const double intake = (shared ? 2.0 : two ? 1.3 : 1.0) *
                                      static_cast<double>((num_k + s - 1) / s) * stage / rate;
                double exchange = s > 1 ? 1.0 + t * G * 512.0 * (s - 1) / s / 30e3 : 0.0;
                if (GATED) exchange = exchange * 1.5 + 0.25 * (s - 1);
                double us = 2.5 + waves * ((two && waves > 1 ? 0.75 : 1.5) + intake + exchange);
                // bound by HBM, two CTAs per SM keep it busier over their ends (8192 x 28672 for
                // one token: 38.5 us, 39.9 us with one)
                const double floor = two ? hbm : 1.04 * hbm;
                if (us < floor) us = floor + 0.02 * us;
                if (us < best.us) {
                    best = p;
                    best.split = s;
                    best.us = us;
                }
            }
        }
    }
    return best;
}

template <bool GATED>
int launch_narrow(const NarrowPlan& plan, Operand a, int a_type, Operand b, Operand b2, int b_type,
                  const Epi& e, int64_t M, int64_t N, int64_t K, cudaStream_t stream) {
    using namespace narrow;
    Shape p = {};
    p.M = static_cast<uint32_t>(M);
    p.N = static_cast<uint32_t>(N);
    p.K = static_cast<uint32_t>(K);
    p.tokens = plan.tokens;
    p.stages = plan.stages;
    p.split = plan.split;
    p.tmem_cols = plan.tmem_cols;
    const uint32_t smem = plan.smem;
    const int64_t blocks = (N + 127) / 128, ytiles = (M + p.tokens - 1) / p.tokens;

    Maps maps = {};
    int st = operand_maps(&maps.x, &maps.sfx, a, M, K, p.tokens);
    if (st) return st;
    st = operand_maps(&maps.w, &maps.sfw, b, N, K, 128);
    if (st) return st;
    if (GATED) {
        st = operand_maps(&maps.w2, &maps.sfw2, b2, N, K, 128);
        if (st) return st;
    }
    st = ptxstd::set_max_dynamic_smem(reinterpret_cast<const void*>(narrow_kernel<GATED>),
                                      227 * 1024 - 1024);
    if (st) return st;
    uint32_t* err = ptxstd::device_error_word();
    if (!err) return PTXSTD_ECUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<uint32_t>(blocks * p.split), static_cast<uint32_t>(ytiles));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, narrow_kernel<GATED>, maps, p, static_cast<uint32_t>(b_type),
                           static_cast<uint32_t>(a_type), e, err) != cudaSuccess)
        return PTXSTD_ECUDA;
    return ptxstd::launch_status();
}

// Estimated time of the wide kernel: a pair's tile costs about 0.31 us per stage while few pairs
// are active, 0.41 us when all are.
double wide_us(int64_t M, int64_t N, int64_t K, bool gated) {
    const int64_t tile_n = gated ? 128 : 256, pairs = ptxstd::sm_count() / 2;
    const int64_t tiles = ((M + 255) / 256) * ((N + tile_n - 1) / tile_n);
    const int64_t waves = (tiles + pairs - 1) / pairs, num_k = (K + BK - 1) / BK;
    return 2.5 + waves * (2.0 + num_k * (tiles > pairs ? 0.41 : 0.31));
}

// The narrow kernel where its estimate is clearly the better one, up to the 1024 rows that the
// estimate was fitted over. Above, always the wide kernel. Both sides there, wide and narrow in us:
// with enough columns the 256-row tiles fill the GPU, and the wide kernel is the faster one
// (2048 x 2048 x 4096 15.9 and 19.0; 2048 x 4096 x 4096 27.9 and 38.1; 4096 x 576 x 7168 24.0 and
// 36.3; gated 2048 x 512 x 4096 14.6 and 15.9). With few columns they do not, and as the wide kernel
// has no split of K a long K is slow (1040 x 128 x 16384 40.4 and 12.2, just above the limit;
// 2048 x 128 x 16384 41.8 and 15.3; 4096 x 128 x 16384 42.7 and 19.6; 2048 x 512 x 16384 43.3 and
// 25.4; 2048 x 1024 x 1024 7.5 and 6.7).
constexpr int64_t kNarrowRows = 1024;

template <bool GATED>
int dispatch(Operand a, int a_type, Operand b, Operand b2, int b_type, const Epi& e, int64_t M,
             int64_t N, int64_t K, cudaStream_t stream) {
    if (M <= kNarrowRows) {
        const NarrowPlan plan = narrow_plan<GATED>(M, N, K);
        if (plan.us < 0.95 * wide_us(M, N, K, GATED))
            return launch_narrow<GATED>(plan, a, a_type, b, b2, b_type, e, M, N, K, stream);
    }
    return launch_wide<GATED>(a, a_type, b, b2, b_type, e, M, N, K, stream);
}

bool bad(const void* p) { return !p || !ptxstd::aligned16(p); }
bool bad_or_null(const void* p) { return p && !ptxstd::aligned16(p); }

int check_common(int a_type, int b_type, int act, int out_type, const Epi& e, int64_t M, int64_t N,
                 int64_t K) {
    if (!mx_type_ok(a_type) || !mx_type_ok(b_type)) return PTXSTD_EINVAL;
    if (act < PTXSTD_ACT_NONE || act > PTXSTD_ACT_GELU_TANH) return PTXSTD_EINVAL;
    if (M <= 0 || N <= 0 || K <= 0 || N % 8 || K % 32) return PTXSTD_EINVAL;
    if (M >= (1ll << 31) || N >= (1ll << 31) || K >= (1ll << 31)) return PTXSTD_EINVAL;
    if (!e.c && !e.q) return PTXSTD_EINVAL;
    if (bad_or_null(e.c) || bad_or_null(e.pre) || bad_or_null(e.up) || bad_or_null(e.bias) ||
        bad_or_null(e.residual) || bad_or_null(e.q))
        return PTXSTD_EINVAL;
    if (e.q && (bad(e.sfq) || N % 32 || (out_type != PTXSTD_MX_E4M3 && out_type != PTXSTD_MX_E5M2)))
        return PTXSTD_EINVAL;
    return PTXSTD_OK;
}

}  // namespace

extern "C" int ptxstd_gemm_mx_epilogue(const uint8_t* d_a, int a_type, const uint8_t* d_sfa,
                                       const uint8_t* d_b, int b_type, const uint8_t* d_sfb,
                                       const uint16_t* d_bias, int act, const uint16_t* d_residual,
                                       uint16_t* d_c, uint16_t* d_pre, int out_type, uint8_t* d_q,
                                       uint8_t* d_sfq, int64_t M, int64_t N, int64_t K,
                                       ptxstd_stream stream) {
    Epi e = {};
    e.bias = d_bias;
    e.residual = d_residual;
    e.c = d_c;
    e.pre = d_pre;
    e.q = d_q;
    e.sfq = d_sfq;
    e.q_type = static_cast<uint32_t>(out_type);
    e.act = static_cast<uint32_t>(act);
    const int st = check_common(a_type, b_type, act, out_type, e, M, N, K);
    if (st) return st;
    if (bad(d_a) || bad(d_sfa) || bad(d_b) || bad(d_sfb)) return PTXSTD_EINVAL;
    return dispatch<false>({d_a, d_sfa}, a_type, {d_b, d_sfb}, {nullptr, nullptr}, b_type, e, M, N,
                           K, static_cast<cudaStream_t>(stream));
}

extern "C" int ptxstd_gemm_mx_gated(const uint8_t* d_a, int a_type, const uint8_t* d_sfa,
                                    const uint8_t* d_wg, const uint8_t* d_sfg, const uint8_t* d_wu,
                                    const uint8_t* d_sfu, int w_type, int act, uint16_t* d_h,
                                    uint16_t* d_gate, uint16_t* d_up, int out_type, uint8_t* d_q,
                                    uint8_t* d_sfq, int64_t M, int64_t F, int64_t K,
                                    ptxstd_stream stream) {
    Epi e = {};
    e.c = d_h;
    e.pre = d_gate;
    e.up = d_up;
    e.q = d_q;
    e.sfq = d_sfq;
    e.q_type = static_cast<uint32_t>(out_type);
    e.act = static_cast<uint32_t>(act);
    const int st = check_common(a_type, w_type, act, out_type, e, M, F, K);
    if (st) return st;
    if (bad(d_a) || bad(d_sfa) || bad(d_wg) || bad(d_sfg) || bad(d_wu) || bad(d_sfu))
        return PTXSTD_EINVAL;
    if ((d_gate == nullptr) != (d_up == nullptr)) return PTXSTD_EINVAL;
    return dispatch<true>({d_a, d_sfa}, a_type, {d_wg, d_sfg}, {d_wu, d_sfu}, w_type, e, M, F, K,
                          static_cast<cudaStream_t>(stream));
}
