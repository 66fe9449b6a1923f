// Products of activations with unquantised fp16 or bf16 weights, dense and grouped by expert:
//
//   y[p][o] = round( act( sum_i x[row(p)][i] * W[e(p)][o][i] + b[e(p)][o] ) + r[p][o] )
//
// Operands of one 16-bit type, fp32 products and sums on the matrix pipe, fp32 epilogue, one
// rounding. A dense product is the case of one expert that holds every position.
//
// One workgroup computes BN weight rows x BM positions. Both panels of a 64-column step (rows of
// 128 bytes) go from memory straight to LDS (16 bytes a lane, no registers) into a ring of S
// stages; the requests for step s+S-1 are issued behind the barrier that opens step s, so S-1
// steps are in flight while one is multiplied. A request instruction fills 8 rows; lane l writes
// LDS unit l of them, and fetches unit (l%8) ^ (l/8) of row l/8: the exclusive-or spreads the
// 16-byte units of 8 consecutive rows over all banks, so that the fragment reads (16 rows, one
// unit each) are free of conflicts, while 8 neighbouring lanes still read 128 contiguous bytes.
//
// Weights are the A operand of v_mfma_f32_16x16x32: lane l ends with four consecutive outputs of
// position l%16. The gated form keeps a wave's gate rows and up rows side by side in the panel,
// so both pre-activations of an output meet in one lane.
#include "product.hpp"

#include <atomic>

namespace aeon355 {

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;           // columns of one pipeline step: 128 bytes of a row
constexpr int kStepBytes = 128;
constexpr int kXcds = 8;
constexpr int kWindowGroup = 8;     // windows that share a pass over the row blocks

struct F16 {
    static __device__ __forceinline__ float4_t mfma(const u32x4_t& a, const u32x4_t& b, const float4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ float widen(uint16_t v) { return half_bits_to_float(v); }
    static __device__ __forceinline__ uint16_t round(float v) { return float_to_half_bits(v); }
};
struct BF16 {
    static __device__ __forceinline__ float4_t mfma(const u32x4_t& a, const u32x4_t& b, const float4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float widen(uint16_t v) {
        return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
    }
    static __device__ __forceinline__ uint16_t round(float v) {  // to nearest even, NaN kept
        return __builtin_bit_cast(uint16_t, static_cast<bf16_t>(v));
    }
};

// Activations in fp32. The clamps are comparisons, not fminf/fmaxf: those return the bound for a
// NaN operand and would turn a NaN pre-activation into a finite value.
__device__ __forceinline__ float activate(int kind, float g, float u, float limit) {
    switch (kind) {
        case AEON_ACT_SILU: return g / (1.0f + expf(-g));
        case AEON_ACT_GELU: return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
        case AEON_ACT_GELU_TANH: {
            const float z = 0.79788456080286536f * (g + 0.044715f * g * g * g);
            return 0.5f * g * (1.0f + tanhf(z));
        }
        case AEON_ACT_SWIGLU: {
            g = g > limit ? limit : g;
            u = u > limit ? limit : (u < -limit ? -limit : u);
            return g / (1.0f + expf(-g)) * u;
        }
        default: return g;
    }
}

// One wave-wide request: 16 bytes of `p` (per lane) to LDS byte `lds` + 16 * lane. Written as
// asm because the compiler makes every later LDS read wait for all requests of the builtin form.
// It has no register result, so nothing is in flight that the compiler could reuse; the waits are
// wait_requests() before the barrier that publishes a stage. M0 is never live across instructions the
// compiler emits: it writes it right before each use.
__device__ __forceinline__ void request_to_lds(const char* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds), "v"(p) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_requests() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "i"(N) : "memory");
}
__device__ __forceinline__ void bare_barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

struct ProductTile {
    int expert, first, count, row_block;  // positions [first, first + count), row block of W
};

// Tile of workgroup b. Workgroups are dealt to the 8 XCDs round robin, so tile numbers are handed
// out in 8 contiguous runs, one per XCD: neighbouring tiles share panels through one L2. Inside an
// expert up to kWindowGroup windows take turns over each row block, a near-square patch of the
// output for the workgroups that run at the same time.
template <int BM>
__device__ __forceinline__ bool find_tile(const ProductArgs& a, int row_blocks, int b, ProductTile* t) {
    const int lane = threadIdx.x & 63;
    int expert = 0, first = 0, held = a.positions, before = 0, windows;
    int total;
    if (a.offsets == nullptr) {
        windows = (held + BM - 1) / BM;
        total = windows * row_blocks;
    }
    const int per = a.offsets == nullptr ? 0 : (a.experts + 63) / 64;
    int mine = 0, upto = 0;
    // list bounds as the caller gave them, held inside [0, positions] and ascending
    auto bound = [&](int e) {
        const int v = a.offsets[e];
        return v < 0 ? 0 : (v > a.positions ? a.positions : v);
    };
    auto windows_of = [&](int e, int* lo, int* n) {
        *lo = bound(e);
        *n = bound(e + 1) - *lo;
        if (*n < 0) *n = 0;
        return (*n + BM - 1) / BM;
    };
    if (a.offsets != nullptr) {
        for (int i = 0; i < per; ++i) {
            const int e = lane * per + i;
            int lo, n;
            if (e < a.experts) mine += windows_of(e, &lo, &n);
        }
        upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(upto, d, 64);
            if (lane >= d) upto += other;
        }
        total = __builtin_amdgcn_readlane(upto, 63) * row_blocks;
    }
    const int run = (total + kXcds - 1) / kXcds;
    const int at = b / kXcds;
    const int tile = (b % kXcds) * run + at;
    if (at >= run || tile >= total) return false;
    if (a.offsets != nullptr) {
        const int lo_tile = (upto - mine) * row_blocks;
        const uint64_t owner = __ballot(tile >= lo_tile && tile < upto * row_blocks);
        const int from = __builtin_ctzll(owner);
        before = upto - mine;
        for (int i = 0; i < per; ++i) {
            const int e = lane * per + i;
            if (e >= a.experts) break;
            int lo, n;
            const int w = windows_of(e, &lo, &n);
            expert = e;
            first = lo;
            held = n;
            if (tile < (before + w) * row_blocks) break;
            before += w;
        }
        expert = __builtin_amdgcn_readlane(expert, from);
        first = __builtin_amdgcn_readlane(first, from);
        held = __builtin_amdgcn_readlane(held, from);
        before = __builtin_amdgcn_readlane(before, from);
        windows = (held + BM - 1) / BM;
    }
    const int u = tile - before * row_blocks;
    const int group = u / (kWindowGroup * row_blocks);
    const int v = u - group * kWindowGroup * row_blocks;
    const int left = windows - group * kWindowGroup;
    const int wide = left < kWindowGroup ? left : kWindowGroup;
    const int window = group * kWindowGroup + v % wide;
    t->expert = expert;
    t->row_block = v / wide;
    t->first = first + window * BM;
    const int rest = held - window * BM;
    t->count = rest < BM ? rest : BM;
    return true;
}

// 16 bytes of a row starting at column c, zeros from column k on. `p` is the row's column 0. The
// address may be off every boundary but the element's; loads of global memory take that.
__device__ __forceinline__ u32x4_t load_columns(const uint16_t* p, int c, int k) {
    typedef u32x4_t __attribute__((aligned(2))) loose_t;
    if (c + 8 <= k) return *reinterpret_cast<const loose_t*>(p + c);
    u32x4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (c + i < k) v[i / 2] |= static_cast<uint32_t>(p[c + i]) << (16 * (i & 1));
    }
    return v;
}

// ALIGNED: x and W start on 16-byte boundaries and their pitches are multiples of 8 elements.
// Otherwise the panels pass through registers, one step ahead of the products (S is 2 then).
template <class T, int BM, int BN, int WAVES_M, int WAVES_N, int S, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void product_kernel(const ProductArgs a) {
    constexpr int WAVES = WAVES_M * WAVES_N;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
    constexpr int TM = WM / 16, TN = WN / 16;
    constexpr int NI = (BM + BN) / 8 / WAVES;  // requests of a wave per step
    constexpr int STAGE = (BM + BN) * kStepBytes;
    static_assert((BM + BN) / 8 % WAVES == 0 && TN % 2 == 0 && BM % 16 == 0 && (ALIGNED || S == 2), "tile");
    extern __shared__ char ring[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_m = wave % WAVES_M, wave_n = wave / WAVES_M;
    const int rows_per_block = a.pair ? BN / 2 : BN;
    const int row_blocks = (a.n + rows_per_block - 1) / rows_per_block;
    ProductTile t;
    if (!find_tile<BM>(a, row_blocks, blockIdx.x, &t)) return;
    const int n0 = t.row_block * rows_per_block;

    int step0 = 0, steps = (a.k + kStep - 1) / kStep;
    if (a.mode == kProductPartial) {
        step0 = blockIdx.y * a.split_steps;
        steps = steps - step0 < a.split_steps ? steps - step0 : a.split_steps;
    }

    // this lane's row of every request: panel rows [0, BN) are weights, [BN, BN + BM) positions;
    // rows past the end repeat the last one and are not stored
    const uint16_t* src[NI];
    const int unit = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (wave * NI + i) * 8 + (lane >> 3);
        if (r < BN) {
            int matrix = 0, row = r;
            if (a.pair) {
                const int q = r % WN;
                matrix = q >= WN / 2;
                row = r / WN * (WN / 2) + q % (WN / 2);
            }
            row += n0;
            row = row < a.n ? row : a.n - 1;
            src[i] = a.w[matrix] + t.expert * a.expert_stride + row * a.w_stride;
        } else {
            int m = r - BN;
            m = t.first + (m < t.count ? m : t.count - 1);
            if (a.rows != nullptr) {
                m = a.rows[m];
                m = m < 0 ? 0 : (m < a.x_rows ? m : a.x_rows - 1);
            }
            src[i] = a.x + m * a.x_stride;
        }
    }

    float4_t acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const uint32_t ring_at = static_cast<uint32_t>(
        reinterpret_cast<size_t>((__attribute__((address_space(3))) char*)ring));
    u32x4_t held[ALIGNED ? 1 : NI];
    auto fetch = [&](int step) {  // a step's share through registers
#pragma unroll
        for (int i = 0; i < NI; ++i) held[ALIGNED ? 0 : i] = load_columns(src[i], (step0 + step) * kStep + unit * 8, a.k);
    };
    auto put = [&](int stage) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            *reinterpret_cast<u32x4_t*>(ring + stage * STAGE + (wave * NI + i) * 1024 + lane * 16) = held[ALIGNED ? 0 : i];
        }
    };
    const int whole = (a.k - step0 * kStep) / kStep;
    const int full = whole < steps ? whole : steps;  // steps before this one have all 64 columns
    auto request = [&](int step, int stage) {
        if (step < full) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                request_to_lds(reinterpret_cast<const char*>(src[i]) + unit * 16 +
                                   static_cast<size_t>(step0 + step) * kStepBytes,
                               ring_at + stage * STAGE + (wave * NI + i) * 1024);
            }
        } else {  // the last columns of a K that is no multiple of 64
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                *reinterpret_cast<u32x4_t*>(ring + stage * STAGE + (wave * NI + i) * 1024 + lane * 16) =
                    load_columns(src[i], (step0 + step) * kStep + unit * 8, a.k);
            }
        }
    };
    const int frag = (lane & 15) * kStepBytes + (((lane >> 4) ^ (lane & 7)) * 16);
    auto multiply = [&](int stage) {
        const char* wp = ring + stage * STAGE + wave_n * WN * kStepBytes;
        const char* xp = ring + stage * STAGE + (BN + wave_m * WM) * kStepBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4_t wf[TN], xf[TM];
#pragma unroll
            for (int i = 0; i < TN; ++i) wf[i] = *reinterpret_cast<const u32x4_t*>(wp + i * 2048 + (frag ^ (h * 64)));
#pragma unroll
            for (int j = 0; j < TM; ++j) xf[j] = *reinterpret_cast<const u32x4_t*>(xp + j * 2048 + (frag ^ (h * 64)));
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = T::mfma(wf[i], xf[j], acc[i][j]);
        }
    };

    if constexpr (ALIGNED) {
#pragma unroll
        for (int s = 0; s < S - 1; ++s) {
            if (s < steps) request(s, s);
        }
        int stage = 0, ahead = S - 1;
        for (int s = 0; s < steps; ++s) {
            // the S-2 younger steps may still be under way, if they are all requests
            if (s + S - 2 < full) wait_requests<(S - 2) * NI>();
            else wait_requests<0>();
            bare_barrier();
            if (s + S - 1 < steps) request(s + S - 1, ahead);
            multiply(stage);
            stage = stage + 1 == S ? 0 : stage + 1;
            ahead = ahead + 1 == S ? 0 : ahead + 1;
        }
    } else {
        if (steps > 0) {
            fetch(0);
            put(0);
        }
        for (int s = 0; s < steps; ++s) {
            __syncthreads();
            if (s + 1 < steps) fetch(s + 1);
            multiply(s & 1);
            if (s + 1 < steps) put((s + 1) & 1);
        }
    }

    // Epilogue: lane holds outputs 4*(lane/16) .. +3 of a 16-row tile for position lane%16.
    const int out0 = n0 + wave_n * (a.pair ? WN / 2 : WN) + (lane >> 4) * 4;
    const int tiles = a.pair ? TN / 2 : TN;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int m = wave_m * WM + j * 16 + (lane & 15);
        if (m >= t.count) continue;
        const int p = t.first + m;
        if (a.rows != nullptr) {
            const int row = a.rows[p];
            if (row < 0 || row >= a.x_rows) continue;
        }
        long draw = 0;
        float draw_weight = 0.0f;
        if (a.mode == kProductDraws) {
            draw = a.draws[p];
            if (draw < 0 || draw >= a.draw_count) continue;
            draw_weight = a.draw_weights[draw];
        }
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int o = out0 + i * 16;
            if (i >= tiles || o >= a.n) break;
            float g[4], u[4];
            if (a.mode == kProductPartial) {
#pragma unroll
                for (int m2 = 0; m2 < 2; ++m2) {
                    if (m2 == 1 && !a.pair) break;
                    float* dst = a.wide + ((static_cast<size_t>(blockIdx.y) * (a.pair + 1) + m2) * a.positions + p) * a.n + o;
                    const float4_t v = m2 == 0 ? acc[i][j] : acc[(i + TN / 2) % TN][j];
                    if (a.n % 4 == 0) {
                        *reinterpret_cast<float4_t*>(dst) = v;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (o + q < a.n) dst[q] = v[q];
                    }
                }
                continue;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bool live = o + q < a.n;
                g[q] = acc[i][j][q];
                if (a.bias[0] != nullptr && live) g[q] += T::widen(a.bias[0][static_cast<size_t>(t.expert) * a.n + o + q]);
                u[q] = 0.0f;
                if (a.pair) {
                    u[q] = acc[(i + TN / 2) % TN][j][q];
                    if (a.bias[1] != nullptr && live) u[q] += T::widen(a.bias[1][static_cast<size_t>(t.expert) * a.n + o + q]);
                }
            }
            if (a.mode == kProductDraws) {
                float* dst = a.wide + static_cast<size_t>(draw) * a.n + o;
                if (a.n % 4 == 0) {
                    *reinterpret_cast<float4_t*>(dst) = float4_t{g[0], g[1], g[2], g[3]} * draw_weight;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (o + q < a.n) dst[q] = g[q] * draw_weight;
                }
                continue;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) g[q] = activate(a.activation, g[q], u[q], a.limit);
            uint16_t* dst = a.y + p * a.y_stride + o;
            const uint16_t* res = a.residual == nullptr ? nullptr : a.residual + p * a.residual_stride + o;
            if (a.vec_out) {
                if (res != nullptr) {
                    const uint2 r = *reinterpret_cast<const uint2*>(res);
                    g[0] += T::widen(r.x & 0xFFFFu);
                    g[1] += T::widen(r.x >> 16);
                    g[2] += T::widen(r.y & 0xFFFFu);
                    g[3] += T::widen(r.y >> 16);
                }
                uint2 v;
                v.x = T::round(g[0]) | (static_cast<uint32_t>(T::round(g[1])) << 16);
                v.y = T::round(g[2]) | (static_cast<uint32_t>(T::round(g[3])) << 16);
                *reinterpret_cast<uint2*>(dst) = v;
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (o + q >= a.n) break;
                    if (res != nullptr) g[q] += T::widen(res[q]);
                    dst[q] = T::round(g[q]);
                }
            }
        }
    }
}

// Joins the shares of K of a dense product, in share order, and applies the epilogue. Four outputs
// a thread.
template <class T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs a, int splits) {
    const int groups = (a.n + 3) / 4;
    const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= static_cast<long>(a.positions) * groups) return;
    const int p = static_cast<int>(at / groups);
    const int o = static_cast<int>(at - static_cast<long>(p) * groups) * 4;
    const int mats = a.pair + 1;
    float v[2][4] = {};
    for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (m >= mats) break;
            const float* src = a.wide + ((static_cast<size_t>(s) * mats + m) * a.positions + p) * a.n + o;
            if (a.n % 4 == 0) {
                const float4_t w = *reinterpret_cast<const float4_t*>(src);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[m][q] += w[q];
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (o + q < a.n) v[m][q] += src[q];
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (o + q >= a.n) break;
        float g = v[0][q], u = v[1][q];
        if (a.bias[0] != nullptr) g += T::widen(a.bias[0][o + q]);
        if (a.pair && a.bias[1] != nullptr) u += T::widen(a.bias[1][o + q]);
        g = activate(a.activation, g, u, a.limit);
        if (a.residual != nullptr) g += T::widen(a.residual[p * a.residual_stride + o + q]);
        a.y[p * a.y_stride + o + q] = T::round(g);
    }
}

// out[t][i] = round(base[t][i] + sum of the token's contributions in slot order). A draw whose id
// is outside [0, experts) holds no contribution and is left out.
template <class T>
__global__ __launch_bounds__(256) void product_combine_kernel(const float* __restrict__ contrib,
                                                              const int32_t* __restrict__ ids, int experts,
                                                              int tokens, int slots, int n, const uint16_t* base,
                                                              long base_stride, uint16_t* out, long out_stride) {
    const int groups = (n + 3) / 4;
    const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= static_cast<long>(tokens) * groups) return;
    const int t = static_cast<int>(at / groups);
    const int o = static_cast<int>(at - static_cast<long>(t) * groups) * 4;
    float v[4] = {};
    if (base != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (o + q < n) v[q] = T::widen(base[t * base_stride + o + q]);
    }
    for (int s = 0; s < slots; ++s) {
        const long draw = static_cast<long>(t) * slots + s;
        const int id = ids[draw];
        if (id < 0 || id >= experts) continue;
        const float* src = contrib + static_cast<size_t>(draw) * n + o;
        if (n % 4 == 0) {
            const float4_t w = __builtin_nontemporal_load(reinterpret_cast<const float4_t*>(src));
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += w[q];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (o + q < n) v[q] += src[q];
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (o + q < n) out[t * out_stride + o + q] = T::round(v[q]);
}

// ---- launches --------------------------------------------------------------------------------

template <class T, int BM, int BN, int WAVES_M, int WAVES_N, int S, bool ALIGNED>
static int launch_tile(const ProductArgs& a, int splits, hipStream_t stream) {
    auto kernel = product_kernel<T, BM, BN, WAVES_M, WAVES_N, S, ALIGNED>;
    constexpr int bytes = S * (BM + BN) * kStepBytes;
    if (bytes > 65536) {
        // more dynamic LDS than the default limit has to be asked for, once per kernel and device
        static std::atomic<uint64_t> raised{0};
        int device = 0;
        AEON_HIP(hipGetDevice(&device));
        const uint64_t bit = 1ull << (device & 63);
        if (device >= 64 || (raised.load(std::memory_order_relaxed) & bit) == 0) {
            AEON_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                         hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            raised.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const long rows = a.pair ? BN / 2 : BN;
    const long row_blocks = (a.n + rows - 1) / rows;
    // an upper bound of the windows: every list that holds something may end in a short one
    long windows = (static_cast<long>(a.positions) + BM - 1) / BM;
    if (a.offsets != nullptr) windows = a.positions / BM + (a.experts < a.positions ? a.experts : a.positions);
    const long grid = (windows * row_blocks + kXcds - 1) / kXcds * kXcds;
    AEON_REQUIRE(grid <= 0x7fffffffL, AEON_ERR_INVALID_ARGUMENT, "product: %ld workgroups are more than one launch holds", grid);
    kernel<<<dim3(static_cast<unsigned>(grid), splits), 64 * WAVES_M * WAVES_N, bytes, stream>>>(a);
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}

template <class T, bool ALIGNED>
static int launch_tiles(int tile, const ProductArgs& a, int splits, hipStream_t stream) {
    if constexpr (ALIGNED) {
        switch (tile) {
            case 16: return launch_tile<T, 16, 64, 1, 2, 7, true>(a, splits, stream);
            case 32: return launch_tile<T, 32, 64, 1, 2, 6, true>(a, splits, stream);
            case 64: return launch_tile<T, 64, 64, 2, 2, 5, true>(a, splits, stream);
            case 128: return launch_tile<T, 128, 128, 2, 2, 2, true>(a, splits, stream);
            default: return launch_tile<T, 256, 256, 2, 4, 2, true>(a, splits, stream);
        }
    } else {
        switch (tile) {
            case 16:
            case 32: return launch_tile<T, 32, 64, 1, 2, 2, false>(a, splits, stream);
            case 64: return launch_tile<T, 64, 64, 2, 2, 2, false>(a, splits, stream);
            default: return launch_tile<T, 128, 128, 2, 2, 2, false>(a, splits, stream);
        }
    }
}

static bool on_boundary(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

static int launch_product(int dtype, int tile, ProductArgs& a, int splits, hipStream_t stream) {
    const bool aligned = on_boundary(a.x, 16) && on_boundary(a.w[0], 16) && on_boundary(a.w[1], 16) &&
                         a.x_stride % 8 == 0 && a.w_stride % 8 == 0 && a.expert_stride % 8 == 0;
    a.vec_out = a.n % 4 == 0 && a.y_stride % 4 == 0 && on_boundary(a.y, 8) && a.residual_stride % 4 == 0 &&
                on_boundary(a.residual, 8);
    if (dtype == AEON_DTYPE_F16) {
        return aligned ? launch_tiles<F16, true>(tile, a, splits, stream) : launch_tiles<F16, false>(tile, a, splits, stream);
    }
    return aligned ? launch_tiles<BF16, true>(tile, a, splits, stream) : launch_tiles<BF16, false>(tile, a, splits, stream);
}

// Positions a tile holds and the shares K is cut into.
struct ProductPlan {
    int tile, splits, split_steps;
};

static ProductPlan plan_linear(const aeon_projection& w, int tokens) {
    const bool pair = w.activation == AEON_ACT_SWIGLU;
    const long n = static_cast<long>(w.out_dim) * (pair ? 2 : 1);
    auto tiles = [&](long bm, long bn) { return (tokens + bm - 1) / bm * ((n + bn - 1) / bn); };
    ProductPlan p{16, 1, 0};
    if (tokens > 16) p.tile = 32;
    if (tokens > 32) p.tile = 64;
    if (tokens > 64 && tiles(128, 128) >= 256) p.tile = 128;
    if (tokens > 128 && tiles(256, 256) >= 192) p.tile = 256;
    const int steps = (w.in_dim + kStep - 1) / kStep;
    const long have = tiles(p.tile, p.tile <= 64 ? 64 : p.tile);
    const long want = p.tile <= 64 ? 512 : 256;
    long splits = want / (have > 0 ? have : 1);
    if (splits > steps / 8) splits = steps / 8;
    if (splits > 16) splits = 16;
    if (splits < 1 || p.tile > 64) splits = 1;
    p.split_steps = static_cast<int>((steps + splits - 1) / splits);
    p.splits = (steps + p.split_steps - 1) / p.split_steps;
    return p;
}

// Experts: by how many positions an expert holds on average.
static int plan_experts(int positions, int experts) {
    const int live = experts < positions ? experts : positions;
    const int mean = positions / (live > 0 ? live : 1);
    return mean <= 8 ? 16 : mean <= 24 ? 32 : mean <= 64 ? 64 : mean <= 256 ? 128 : 256;
}

static int check_projection(const aeon_projection* w, const char* who) {
    AEON_REQUIRE(w != nullptr, AEON_ERR_INVALID_ARGUMENT, "%s: null projection", who);
    AEON_REQUIRE(w->dtype == AEON_DTYPE_F16 || w->dtype == AEON_DTYPE_BF16, AEON_ERR_INVALID_ARGUMENT,
                 "%s: unknown dtype %d", who, w->dtype);
    AEON_REQUIRE(w->in_dim > 0 && w->out_dim > 0 && w->in_dim <= (1 << 24) && w->out_dim <= (1 << 24),
                 AEON_ERR_INVALID_ARGUMENT, "%s: bad shape (in_dim=%d out_dim=%d)", who, w->in_dim, w->out_dim);
    AEON_REQUIRE(w->weight_stride >= w->in_dim, AEON_ERR_INVALID_ARGUMENT, "%s: weight rows of %ld elements overlap (in_dim=%d)",
                 who, w->weight_stride, w->in_dim);
    AEON_REQUIRE(w->activation >= AEON_ACT_NONE && w->activation <= AEON_ACT_SWIGLU, AEON_ERR_INVALID_ARGUMENT,
                 "%s: unknown activation %d", who, w->activation);
    AEON_REQUIRE(w->d_weight != nullptr, AEON_ERR_INVALID_ARGUMENT, "%s: null weight", who);
    const bool pair = w->activation == AEON_ACT_SWIGLU;
    AEON_REQUIRE(pair == (w->d_weight_up != nullptr), AEON_ERR_INVALID_ARGUMENT,
                 "%s: a second weight matrix belongs to the gated activation, and to no other", who);
    AEON_REQUIRE(pair || w->d_bias_up == nullptr, AEON_ERR_INVALID_ARGUMENT,
                 "%s: a second bias belongs to the gated activation", who);
    AEON_REQUIRE(!pair || w->swiglu_limit > 0.0f, AEON_ERR_INVALID_ARGUMENT,
                 "%s: swiglu_limit must be positive (infinity for no clamp)", who);
    AEON_REQUIRE(on_boundary(w->d_weight, 2) && on_boundary(w->d_weight_up, 2) && on_boundary(w->d_bias, 2) &&
                     on_boundary(w->d_bias_up, 2),
                 AEON_ERR_INVALID_ARGUMENT, "%s: a 16-bit operand starts on an odd address", who);
    return AEON_OK;
}

static ProductArgs projection_args(const aeon_projection& w) {
    ProductArgs a{};
    a.w[0] = static_cast<const uint16_t*>(w.d_weight);
    a.w[1] = static_cast<const uint16_t*>(w.d_weight_up);
    a.w_stride = w.weight_stride;
    a.bias[0] = static_cast<const uint16_t*>(w.d_bias);
    a.bias[1] = static_cast<const uint16_t*>(w.d_bias_up);
    a.n = w.out_dim;
    a.k = w.in_dim;
    a.pair = w.activation == AEON_ACT_SWIGLU;
    a.activation = w.activation;
    a.limit = w.swiglu_limit;
    return a;
}

static int check_experts(const aeon_projection& w, int experts, long expert_stride, int positions, const char* who) {
    AEON_REQUIRE(experts > 0 && experts <= 1024, AEON_ERR_INVALID_ARGUMENT, "%s: expert count out of range (%d)", who, experts);
    AEON_REQUIRE(positions >= 0, AEON_ERR_INVALID_ARGUMENT, "%s: negative count", who);
    AEON_REQUIRE(expert_stride >= (w.out_dim - 1) * w.weight_stride + w.in_dim, AEON_ERR_INVALID_ARGUMENT,
                 "%s: expert matrices %ld elements apart overlap", who, expert_stride);
    return AEON_OK;
}

static size_t linear_workspace(const aeon_projection& w, int tokens, const ProductPlan& p) {
    if (p.splits == 1) return 0;
    return static_cast<size_t>(p.splits) * (w.activation == AEON_ACT_SWIGLU ? 2 : 1) * tokens * w.out_dim * sizeof(float);
}

}  // namespace aeon355

using namespace aeon355;

extern "C" size_t aeon_linear_workspace_bytes(const aeon_projection* projection, int tokens) {
    if (check_projection(projection, "aeon_linear_workspace_bytes") != AEON_OK || tokens <= 0) return 0;
    return linear_workspace(*projection, tokens, plan_linear(*projection, tokens));
}

extern "C" int aeon_linear(const aeon_projection* projection, const void* d_x, long x_stride, int tokens,
                           const void* d_residual, long residual_stride, void* d_y, long y_stride,
                           void* d_workspace, size_t workspace_bytes, void* stream) {
    const char* who = "aeon_linear";
    if (int rc = check_projection(projection, who)) return rc;
    const aeon_projection& w = *projection;
    AEON_REQUIRE(tokens >= 0, AEON_ERR_INVALID_ARGUMENT, "%s: negative token count", who);
    if (tokens == 0) return AEON_OK;
    AEON_REQUIRE(d_x && d_y, AEON_ERR_INVALID_ARGUMENT, "%s: null buffer", who);
    AEON_REQUIRE(on_boundary(d_x, 2) && on_boundary(d_y, 2) && on_boundary(d_residual, 2), AEON_ERR_INVALID_ARGUMENT,
                 "%s: a 16-bit operand starts on an odd address", who);
    AEON_REQUIRE(x_stride >= w.in_dim && y_stride >= w.out_dim && (d_residual == nullptr || residual_stride >= w.out_dim),
                 AEON_ERR_INVALID_ARGUMENT, "%s: bad row pitch (x %ld, residual %ld, y %ld)", who, x_stride,
                 residual_stride, y_stride);
    AEON_REQUIRE(d_y != d_x && d_y != w.d_weight && d_y != w.d_weight_up, AEON_ERR_INVALID_ARGUMENT,
                 "%s: the output must not alias the activations or the weights", who);
    AEON_REQUIRE(d_y != d_residual || y_stride == residual_stride, AEON_ERR_INVALID_ARGUMENT,
                 "%s: an output on the residual needs the residual's row pitch", who);
    const ProductPlan plan = plan_linear(w, tokens);
    const size_t need = linear_workspace(w, tokens, plan);
    AEON_REQUIRE(workspace_bytes >= need && (need == 0 || (d_workspace != nullptr && on_boundary(d_workspace, 16))),
                 AEON_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes on a 16-byte boundary (%zu given)", who, need,
                 workspace_bytes);
    ProductArgs a = projection_args(w);
    a.x = static_cast<const uint16_t*>(d_x);
    a.x_stride = x_stride;
    a.x_rows = tokens;
    a.positions = tokens;
    a.residual = static_cast<const uint16_t*>(d_residual);
    a.residual_stride = d_residual != nullptr ? residual_stride : 0;
    a.y = static_cast<uint16_t*>(d_y);
    a.y_stride = y_stride;
    if (plan.splits == 1) return launch_product(w.dtype, plan.tile, a, 1, as_stream(stream));
    a.mode = kProductPartial;
    a.wide = static_cast<float*>(d_workspace);
    a.split_steps = plan.split_steps;
    if (int rc = launch_product(w.dtype, plan.tile, a, plan.splits, as_stream(stream))) return rc;
    const long threads = static_cast<long>(tokens) * ((w.out_dim + 3) / 4);
    const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
    if (w.dtype == AEON_DTYPE_F16) product_join_kernel<F16><<<blocks, 256, 0, as_stream(stream)>>>(a, plan.splits);
    else product_join_kernel<BF16><<<blocks, 256, 0, as_stream(stream)>>>(a, plan.splits);
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}

extern "C" int aeon_expert_linear(const aeon_projection* projection, int experts, long expert_stride,
                                  const void* d_x, long x_stride, int x_rows, const int32_t* d_expert_offsets,
                                  const int32_t* d_row_indices, int positions, void* d_y, long y_stride,
                                  void* stream) {
    const char* who = "aeon_expert_linear";
    if (int rc = check_projection(projection, who)) return rc;
    const aeon_projection& w = *projection;
    if (int rc = check_experts(w, experts, expert_stride, positions, who)) return rc;
    if (positions == 0) return AEON_OK;
    AEON_REQUIRE(d_x && d_expert_offsets && d_y, AEON_ERR_INVALID_ARGUMENT, "%s: null buffer", who);
    AEON_REQUIRE(x_rows > 0 && (d_row_indices != nullptr || x_rows >= positions), AEON_ERR_INVALID_ARGUMENT,
                 "%s: %d rows for %d positions", who, x_rows, positions);
    AEON_REQUIRE(on_boundary(d_x, 2) && on_boundary(d_y, 2) && on_boundary(d_expert_offsets, 4) && on_boundary(d_row_indices, 4),
                 AEON_ERR_INVALID_ARGUMENT, "%s: an operand starts off its element's boundary", who);
    AEON_REQUIRE(x_stride >= w.in_dim && y_stride >= w.out_dim, AEON_ERR_INVALID_ARGUMENT, "%s: bad row pitch (x %ld, y %ld)",
                 who, x_stride, y_stride);
    AEON_REQUIRE(d_y != d_x && d_y != w.d_weight && d_y != w.d_weight_up, AEON_ERR_INVALID_ARGUMENT,
                 "%s: the output must not alias the activations or the weights", who);
    ProductArgs a = projection_args(w);
    a.expert_stride = expert_stride;
    a.x = static_cast<const uint16_t*>(d_x);
    a.x_stride = x_stride;
    a.rows = d_row_indices;
    a.x_rows = x_rows;
    a.offsets = d_expert_offsets;
    a.experts = experts;
    a.positions = positions;
    a.y = static_cast<uint16_t*>(d_y);
    a.y_stride = y_stride;
    return launch_product(w.dtype, plan_experts(positions, experts), a, 1, as_stream(stream));
}

extern "C" size_t aeon_expert_combine_workspace_bytes(const aeon_projection* projection, int tokens, int slots) {
    if (check_projection(projection, "aeon_expert_combine_workspace_bytes") != AEON_OK || tokens <= 0 || slots <= 0) return 0;
    return static_cast<size_t>(tokens) * slots * projection->out_dim * sizeof(float);
}

extern "C" int aeon_expert_combine(const aeon_projection* projection, int experts, long expert_stride,
                                   const void* d_h, long h_stride, const int32_t* d_expert_offsets,
                                   const int32_t* d_draw_indices, const int32_t* d_topk_ids,
                                   const float* d_topk_weights, int tokens, int slots, const void* d_base,
                                   long base_stride, void* d_out, long out_stride, void* d_workspace,
                                   size_t workspace_bytes, void* stream) {
    const char* who = "aeon_expert_combine";
    if (int rc = check_projection(projection, who)) return rc;
    const aeon_projection& w = *projection;
    AEON_REQUIRE(w.activation == AEON_ACT_NONE, AEON_ERR_INVALID_ARGUMENT, "%s: takes no activation", who);
    AEON_REQUIRE(tokens >= 0 && slots > 0 && static_cast<long>(tokens) * slots <= 0x7fffffffL, AEON_ERR_INVALID_ARGUMENT,
                 "%s: bad draw shape (tokens=%d slots=%d)", who, tokens, slots);
    if (int rc = check_experts(w, experts, expert_stride, tokens * slots, who)) return rc;
    if (tokens == 0) return AEON_OK;
    AEON_REQUIRE(d_h && d_expert_offsets && d_draw_indices && d_topk_ids && d_topk_weights && d_out, AEON_ERR_INVALID_ARGUMENT,
                 "%s: null buffer", who);
    AEON_REQUIRE(on_boundary(d_h, 2) && on_boundary(d_out, 2) && on_boundary(d_base, 2) && on_boundary(d_expert_offsets, 4) &&
                     on_boundary(d_draw_indices, 4) && on_boundary(d_topk_ids, 4) && on_boundary(d_topk_weights, 4),
                 AEON_ERR_INVALID_ARGUMENT, "%s: an operand starts off its element's boundary", who);
    AEON_REQUIRE(h_stride >= w.in_dim && out_stride >= w.out_dim && (d_base == nullptr || base_stride >= w.out_dim),
                 AEON_ERR_INVALID_ARGUMENT, "%s: bad row pitch (h %ld, base %ld, out %ld)", who, h_stride, base_stride, out_stride);
    AEON_REQUIRE(d_out != d_h && d_out != w.d_weight, AEON_ERR_INVALID_ARGUMENT,
                 "%s: the output must not alias the hidden rows or the weights", who);
    AEON_REQUIRE(d_out != d_base || out_stride == base_stride, AEON_ERR_INVALID_ARGUMENT,
                 "%s: an output on the base needs the base's row pitch", who);
    const size_t need = aeon_expert_combine_workspace_bytes(projection, tokens, slots);
    AEON_REQUIRE(workspace_bytes >= need && d_workspace != nullptr && on_boundary(d_workspace, 16), AEON_ERR_INVALID_ARGUMENT,
                 "%s: needs a workspace of %zu bytes on a 16-byte boundary (%zu given)", who, need, workspace_bytes);
    ProductArgs a = projection_args(w);
    a.expert_stride = expert_stride;
    a.x = static_cast<const uint16_t*>(d_h);
    a.x_stride = h_stride;
    a.x_rows = tokens * slots;
    a.offsets = d_expert_offsets;
    a.experts = experts;
    a.positions = tokens * slots;
    a.mode = kProductDraws;
    a.wide = static_cast<float*>(d_workspace);
    a.draws = d_draw_indices;
    a.draw_weights = d_topk_weights;
    a.draw_count = tokens * slots;
    if (int rc = launch_product(w.dtype, plan_experts(a.positions, experts), a, 1, as_stream(stream))) return rc;
    const long threads = static_cast<long>(tokens) * ((w.out_dim + 3) / 4);
    AEON_REQUIRE((threads + 255) / 256 <= 0x7fffffffL, AEON_ERR_INVALID_ARGUMENT, "%s: too many outputs for one launch", who);
    const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
    const auto* base = static_cast<const uint16_t*>(d_base);
    auto* out = static_cast<uint16_t*>(d_out);
    if (w.dtype == AEON_DTYPE_F16) {
        product_combine_kernel<F16><<<blocks, 256, 0, as_stream(stream)>>>(a.wide, d_topk_ids, experts, tokens, slots, w.out_dim,
                                                                          base, base_stride, out, out_stride);
    } else {
        product_combine_kernel<BF16><<<blocks, 256, 0, as_stream(stream)>>>(a.wide, d_topk_ids, experts, tokens, slots, w.out_dim,
                                                                           base, base_stride, out, out_stride);
    }
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}
