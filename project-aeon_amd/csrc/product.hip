// Products of activations with unquantised fp16 or bf16 weights, dense and grouped by expert:
//
//   y[p][o] = round( act( sum_i x[row(p)][i] * W[e(p)][o][i] + b[e(p)][o] ) + r[p][o] )
//
// Operands of one 16-bit type, fp32 products and sums on the matrix pipe, fp32 epilogue, one
// rounding. A dense product is the case of one expert that holds every position.
//
// One workgroup computes BN weight rows x BM positions. Both panels of a 64-column step (rows of
// 128 bytes) go from memory straight to LDS (16 bytes a lane, no registers) into a ring of S
// stages. A request instruction fills 8 rows; lane l writes LDS unit l of them, and fetches unit
// (l%8) ^ (l/8) of row l/8: the exclusive-or spreads the 16-byte units of 8 consecutive rows over
// all banks, so that the fragment reads (16 rows, one unit each) are free of conflicts, while 8
// neighbouring lanes still read 128 contiguous bytes.
//
// Weights are the A operand of v_mfma_f32_16x16x32: a lane ends with four rows of each 16-row tile
// for position l%16. The gated form keeps a wave's gate rows and up rows side by side in the panel,
// so both pre-activations of an output meet in one lane.
//
// What bounds it, by tile (positions x rows; chosen by plan_linear and plan_experts):
//   4 x any    launch and a trip to memory (1 token, 4096 -> 256: 3.4 us), and the FMAs from two positions on
//   16..64     the weight stream while it is long: 7.1 TB/s over 12.9 GB (64 tokens, 256 experts); in
//              short products a workgroup's own start and end, and with 64 positions the bytes under way:
//              half of the ring holds positions (64 tokens, 7168 -> 7168: 224 workgroups ask for 7 MB of
//              weights ahead, and 103 MB take 24 us)
//   128, 256   the matrix pipe: a 256 x 256 x 64 step takes 1.36 us where the panels are in L2, 1.58
//              PFLOP/s; 2.07 us where every weight panel is one workgroup's own and comes from
//              HBM, because a CU's 64 KB a step then wait for misses of twice the latency
#include "product.hpp"

#include <atomic>
#include <type_traits>

namespace aeon355 {

typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <int N>
using C = std::integral_constant<int, N>;

constexpr int kStep = 64;           // columns of one pipeline step: 128 bytes of a row
constexpr int kStepBytes = 128;
constexpr int kXcds = 8;
constexpr int kXcdCus = 32;
constexpr int kWindowGroup = 8;     // windows that share a pass over the row blocks

struct F16 {
    static __device__ __forceinline__ float4_t mfma(const u32x4_t& a, const u32x4_t& b, const float4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
    }
    static __device__ __forceinline__ float widen(uint16_t v) { return half_bits_to_float(v); }
    static __device__ __forceinline__ uint16_t round(float v) { return float_to_half_bits(v); }
    static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, half2_t{static_cast<half_t>(lo), static_cast<half_t>(hi)});
    }
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
    static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<bf16_t>(lo), static_cast<bf16_t>(hi)});
    }
};

// 1 / (1 + exp(-z)): the exponential by the hardware's power of two. z * log2(e) is rounded to 24
// bits, which shifts the exponential by at most |z| * 2^-24 of itself; the result is rounded to 11 bits
// or fewer. Saturates to 0 and 1 without NaN.
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

// Activations in fp32, in place on N values. gelu takes 1 + erf(z) as erfc(-z), and gelu_tanh
// (1 + tanh z) / 2 as sigmoid(2z): without the cancellation at large negative z. The clamps are comparisons, not fminf/fmaxf: those return
// the bound for a NaN operand and would turn a NaN pre-activation into a finite value.
template <int N>
__device__ __forceinline__ void activate(int kind, float (&g)[N], const float (&u)[N], float limit) {
    switch (kind) {
        case AEON_ACT_SILU:
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] *= sigmoid(g[i]);
            break;
        case AEON_ACT_GELU:
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] *= 0.5f * erfcf(g[i] * -0.70710678118654752f);
            break;
        case AEON_ACT_GELU_TANH:
#pragma unroll
            for (int i = 0; i < N; ++i)
                g[i] *= sigmoid(2.0f * 0.79788456080286536f * (g[i] + 0.044715f * g[i] * g[i] * g[i]));
            break;
        case AEON_ACT_SWIGLU:
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = g[i] > limit ? limit : g[i];
                const float y = u[i] > limit ? limit : (u[i] < -limit ? -limit : u[i]);
                g[i] = x * sigmoid(x) * y;
            }
            break;
        default: break;
    }
}

// One wave-wide request: 16 bytes of `p` (per lane) to LDS byte `lds` + 16 * lane. Written as
// asm because the compiler makes every later LDS read wait for all requests of the builtin form.
// It has no register result, so nothing is in flight that the compiler could reuse; the waits are
// wait_requests() before the barrier that publishes a stage. M0 is never live across instructions the
// compiler emits: it writes it right before each use.
// STREAM: the bytes are read by this workgroup alone and should not push others out of the caches.
template <bool STREAM>
__device__ __forceinline__ void request_to_lds(const char* p, uint32_t lds) {
    if constexpr (STREAM) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
                     :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p) : "memory");
    } else {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                     :: "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p) : "memory");
    }
}
template <int N>
__device__ __forceinline__ void wait_requests() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "i"(N) : "memory");
}
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void bare_barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

struct ProductTile {
    int expert, first, count, row_block;  // positions [first, first + count), row block of W
    bool only;                            // no other window of the list reads these rows
};

// List of expert e as the caller gave it, held inside [0, positions].
__device__ __forceinline__ int list_of(const ProductArgs& a, int e, int* first) {
    auto bound = [&](int i) {
        const int v = a.offsets[i];
        return v < 0 ? 0 : (v > a.positions ? a.positions : v);
    };
    *first = bound(e);
    const int n = bound(e + 1) - *first;
    return n > 0 ? n : 0;
}

// Window and row block of a list's tile u: up to kWindowGroup windows take turns over each row
// block, a near-square patch of the output for the workgroups that run at the same time.
__device__ __forceinline__ void patch_of(int u, int windows, int row_blocks, int* window, int* row_block) {
    const int group = u / (kWindowGroup * row_blocks);
    const int v = u - group * kWindowGroup * row_blocks;
    const int left = windows - group * kWindowGroup;
    const int wide = left < kWindowGroup ? left : kWindowGroup;
    *window = group * kWindowGroup + v % wide;
    *row_block = v / wide;
}

// Tile of workgroup b. Workgroups are dealt to the 8 XCDs round robin, so tiles are handed out in 8
// contiguous runs, one per XCD: neighbouring tiles share panels through one L2.
// TURNS: one workgroup fills a CU, and a tile with at most half of its positions is cheaper. Where at
// most half of the CUs would have a tile in an XCD's last round, a dense product's tiles of that round
// are cut in two (the second part of a short one is empty).
template <int BM, bool TURNS>
__device__ __forceinline__ bool find_tile(const ProductArgs& a, int row_blocks, int b, ProductTile* t) {
    const int lane = threadIdx.x & 63;
    const bool lists = a.offsets != nullptr;
    const int per = lists ? (a.experts + 63) / 64 : 0;  // experts a lane looks after
    int mine = 0, upto = 0, total;
    if (!lists) {
        total = (a.positions + BM - 1) / BM * row_blocks;
    } else {
        for (int e = lane * per; e < (lane + 1) * per && e < a.experts; ++e) {
            int first;
            mine += (list_of(a, e, &first) + BM - 1) / BM;
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
    int at = b / kXcds, half = -1;
    if (TURNS && !lists) {
        const int last = run % kXcdCus;
        if (last <= kXcdCus / 2 && at >= run - last) {
            half = (at - (run - last)) & 1;
            at = run - last + (at - (run - last)) / 2;
        }
    }
    const int tile = (b % kXcds) * run + at;
    if (at >= run || tile >= total) return false;
    int expert = 0, first = 0, held = a.positions, before = 0;
    if (lists) {
        before = upto - mine;
        const uint64_t owner = __ballot(tile >= before * row_blocks && tile < upto * row_blocks);
        if (owner == 0) return false;  // only where the bounds do not ascend
        const int from = __builtin_ctzll(owner);
        for (int e = lane * per; e < (lane + 1) * per && e < a.experts; ++e) {
            expert = e;
            held = list_of(a, e, &first);
            const int w = (held + BM - 1) / BM;
            if (tile < (before + w) * row_blocks) break;
            before += w;
        }
        expert = __builtin_amdgcn_readlane(expert, from);
        first = __builtin_amdgcn_readlane(first, from);
        held = __builtin_amdgcn_readlane(held, from);
        before = __builtin_amdgcn_readlane(before, from);
    }
    const int windows = (held + BM - 1) / BM;
    const int u = tile - before * row_blocks;
    if (u < 0 || u >= windows * row_blocks) return false;  // only where they do not, and the sums wrapped
    int window;
    patch_of(u, windows, row_blocks, &window, &t->row_block);
    t->expert = expert;
    t->only = windows == 1;
    t->first = first + window * BM;
    t->count = held - window * BM < BM ? held - window * BM : BM;
    if (half >= 0) {
        t->first += half * (BM / 2);
        t->count -= half * (BM / 2);
        if (half == 0 && t->count > BM / 2) t->count = BM / 2;
    }
    return t->count > 0;
}

// 16 bytes of a row starting at column c, zeros from column k on. `p` is the row's column 0; nothing
// outside the row's k columns is read. The address may be off every boundary but the element's; loads of
// global memory take that.
__device__ __forceinline__ u32x4_t load_columns(const uint16_t* p, int c, int k) {
    typedef u32x4_t __attribute__((aligned(2))) loose_t;
    const AEON_GLOBAL uint16_t* row = as_global<uint16_t>(p);
    if (c + 8 <= k) return *reinterpret_cast<const AEON_GLOBAL loose_t*>(row + c);
    unsigned __int128 v = 0;
    if (c < k && k >= 8) {  // the row's last eight values, the ones before column c shifted out
        v = __builtin_bit_cast(unsigned __int128, *reinterpret_cast<const AEON_GLOBAL loose_t*>(row + k - 8));
        v >>= (c + 8 - k) * 16;
    } else {
#pragma unroll 1
        for (int i = k - 1; i >= c; --i) v = v << 16 | row[i];
    }
    return __builtin_bit_cast(u32x4_t, v);
}

// Four outputs o .. o+3 of a row of n, fp32 or one 16-bit type, at any element's alignment (global
// memory takes that); the ones past the row's end are zeros, or not written.
__device__ __forceinline__ void store_wide(float* p, const float4_t& v, int o, int n) {
    typedef float4_t __attribute__((aligned(4))) loose_t;
    if (o + 4 <= n) {
        *reinterpret_cast<loose_t*>(p) = v;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (o + q < n) p[q] = v[q];
    }
}
__device__ __forceinline__ float4_t load_wide(const float* p, int o, int n) {
    typedef float4_t __attribute__((aligned(4))) loose_t;
    if (o + 4 <= n) return __builtin_nontemporal_load(reinterpret_cast<const loose_t*>(p));
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (o + q < n) v[q] = p[q];
    return v;
}
template <class T>
__device__ __forceinline__ float4_t load_narrow(const uint16_t* p, int o, int n) {
    typedef u32x2_t __attribute__((aligned(2))) loose_t;
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (o + 4 <= n) {
        const u32x2_t r = *reinterpret_cast<const loose_t*>(p);
        v = float4_t{T::widen(r[0] & 0xFFFFu), T::widen(r[0] >> 16), T::widen(r[1] & 0xFFFFu), T::widen(r[1] >> 16)};
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (o + q < n) v[q] = T::widen(p[q]);
    }
    return v;
}
// The one rounding.
template <class T>
__device__ __forceinline__ void store_narrow(uint16_t* p, const float4_t& v, int o, int n) {
    typedef u32x2_t __attribute__((aligned(2))) loose_t;
    if (o + 4 <= n) {
        *reinterpret_cast<loose_t*>(p) = u32x2_t{T::round2(v[0], v[1]), T::round2(v[2], v[3])};
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (o + q < n) p[q] = T::round(v[q]);
    }
}

// V (4 or 8) of a row's outputs in one 16-bit type, packed in pairs.
template <class T, int V>
struct Narrow {
    typedef uint32_t packed_t __attribute__((ext_vector_type(V / 2)));
    typedef packed_t __attribute__((aligned(2))) loose_t;
    packed_t p;
    __device__ __forceinline__ float value(int k) const { return T::widen(static_cast<uint16_t>(p[k / 2] >> (16 * (k & 1)))); }
    __device__ __forceinline__ void round(const float (&v)[V]) {
#pragma unroll
        for (int k = 0; k < V; k += 2) p[k / 2] = T::round2(v[k], v[k + 1]);
    }
    __device__ __forceinline__ void load(const uint16_t* at, int o, int n) {
        if (o + V <= n) {
            p = *reinterpret_cast<const loose_t*>(at);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (k % 2 == 0) p[k / 2] = 0;
                if (o + k < n) p[k / 2] |= static_cast<uint32_t>(at[k]) << (16 * (k & 1));
            }
        }
    }
    __device__ __forceinline__ void store(uint16_t* at, int o, int n) const {
        if (o + V <= n) {
            *reinterpret_cast<loose_t*>(at) = p;
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (o + k < n) at[k] = static_cast<uint16_t>(p[k / 2] >> (16 * (k & 1)));
        }
    }
};

// Output of row r of a wave's ROWS panel rows of one matrix: in 32 rows the outputs of two 16-row tiles
// are dealt out so that a lane's four rows of one tile and of the other follow each other.
template <int ROWS>
__device__ __forceinline__ int output_of(int r) {
    return ROWS < 32 ? r : r / 32 * 32 + r % 16 / 4 * 8 + r % 32 / 16 * 4 + r % 4;
}

// The tile that fills a CU is run by waves that take turns (below).
constexpr bool takes_turns(int bm, bool aligned) { return aligned && bm == 256; }

// ALIGNED: every row of x and W starts on a 4-byte boundary, which is what vector memory asks for.
// Otherwise the panels pass through registers, one step ahead of the products (S is 2 then).
template <class T, int BM, int BN, int WAVES_M, int WAVES_N, int S, bool ALIGNED>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N) void product_kernel(const ProductArgs a) {
    constexpr int WAVES = WAVES_M * WAVES_N;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
    constexpr int TM = WM / 16, TN = WN / 16;
    constexpr int NW = BN / 8 / WAVES, NI = NW + BM / 8 / WAVES;  // requests of a wave per step: weights, then positions
    constexpr int STAGE = (BM + BN) * kStepBytes;  // of the ring: weight rows, then positions
    constexpr bool TURNS = takes_turns(BM, ALIGNED);
    static_assert(!TURNS || (BN == 256 && WAVES == 8 && S == 2 && TM == 8 && TN == 4), "the schedule of the waves that take turns");
    static_assert(BN / 8 % WAVES == 0 && BM / 8 % WAVES == 0 && TN % 2 == 0 && BM % 16 == 0 && (ALIGNED || S == 2), "tile");
    extern __shared__ char ring[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_m = wave % WAVES_M, wave_n = wave / WAVES_M;
    const int rows_per_block = a.pair ? BN / 2 : BN;
    const int row_blocks = (a.n + rows_per_block - 1) / rows_per_block;
    ProductTile t;
    if (!find_tile<BM, TURNS>(a, row_blocks, blockIdx.x, &t)) return;
    const int n0 = t.row_block * rows_per_block;

    int step0 = 0, steps = (a.k + kStep - 1) / kStep;
    if (a.mode == kProductPartial) {
        step0 = blockIdx.y * a.split_steps;
        steps = steps - step0 < a.split_steps ? steps - step0 : a.split_steps;
    }

    // First panel row of a wave's request i. The kernel whose waves take turns asks for a step in
    // four parts, two requests a wave each: the first half of every wave's weight rows, the first
    // half of its positions, and the second halves.
    auto panel_row = [&](int i) __attribute__((always_inline)) {
        if constexpr (TURNS) {
            const int q = (wave * 2 + (i & 1)) * 8;
            const int half = i / 4;
            return (i / 2) % 2 == 0 ? q / (WN / 2) * WN + half * (WN / 2) + q % (WN / 2)
                                    : BN + q / (WM / 2) * WM + half * (WM / 2) + q % (WM / 2);
        } else {
            return i < NW ? (wave * NW + i) * 8 : BN + (wave * (NI - NW) + i - NW) * 8;
        }
    };
    // Position a panel row holds. Where waves take turns, a wave's first half of positions lies in the
    // tile's first half: a tile with no more than that many live ones skips the second halves.
    auto position_of = [&](int r) __attribute__((always_inline)) {
        return TURNS ? r % WM / (WM / 2) * (BM / 2) + r / WM * (WM / 2) + r % (WM / 2) : r;
    };
    // this lane's row of every request: panel rows [0, BN) are weights, [BN, BN + BM) positions;
    // rows past the end repeat the last one and are not stored
    const uint16_t* src[NI];
    const int unit = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = panel_row(i) + (lane >> 3);
        if (r < BN) {
            int matrix = 0, row;
            if (a.pair) {  // a wave's first half are gate rows, its second half up rows
                const int q = r % WN;
                matrix = q >= WN / 2;
                row = r / WN * (WN / 2) + output_of<WN / 2>(q % (WN / 2));
            } else {
                row = r / WN * WN + output_of<WN>(r % WN);
            }
            row += n0;
            row = row < a.n ? row : a.n - 1;
            src[i] = a.w[matrix] + t.expert * a.expert_stride + row * a.w_stride;
        } else {
            int m = position_of(r - BN);
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
    const int whole = (a.k - step0 * kStep) / kStep;
    const int full = whole < steps ? whole : steps;  // steps of 64 columns; a shorter one may follow
    // requests [first, first + count) of a whole step
    auto request = [&](int step, int stage, auto first, auto count, auto stream) __attribute__((always_inline)) {
#pragma unroll
        for (int i = first; i < first + count; ++i) {
            const char* p = reinterpret_cast<const char*>(src[i]) + unit * 16 +
                            static_cast<size_t>(step0 + step) * kStepBytes;
            const uint32_t lds = ring_at + stage * STAGE + panel_row(i) * kStepBytes;
            if (stream && i < NW) request_to_lds<true>(p, lds);
            else request_to_lds<false>(p, lds);
        }
    };
    // a step through registers, columns from K on as zeros
    u32x4_t held[NI];
    auto fetch = [&](int step) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i) held[i] = load_columns(src[i], (step0 + step) * kStep + unit * 8, a.k);
    };
    auto put = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
            *reinterpret_cast<u32x4_t*>(ring + stage * STAGE + panel_row(i) * kStepBytes + lane * 16) = held[i];
    };
    const int frag = (lane & 15) * kStepBytes + (((lane >> 4) ^ (lane & 7)) * 16);
    struct Fragments {
        u32x4_t w[2][TN], x[2][TM];  // [columns 32h ..][tile]
    };
    auto read_step = [&](Fragments& f, int stage) __attribute__((always_inline)) {
        const char* wp = ring + stage * STAGE + wave_n * WN * kStepBytes;
        const char* xp = ring + stage * STAGE + (BN + wave_m * WM) * kStepBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < TN; ++i) f.w[h][i] = *reinterpret_cast<const u32x4_t*>(wp + i * 2048 + (frag ^ (h * 64)));
#pragma unroll
            for (int j = 0; j < TM; ++j) f.x[h][j] = *reinterpret_cast<const u32x4_t*>(xp + j * 2048 + (frag ^ (h * 64)));
        }
    };
    auto multiply = [&](const Fragments& f) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = T::mfma(f.w[h][i], f.x[h][j], acc[i][j]);
    };

    if constexpr (TURNS) {
        // Two waves share a SIMD; they take turns at its matrix pipe. A step is two parts of 32
        // MFMAs a wave, one for each half of its positions, and a part a fetch (LDS reads, requests)
        // and a multiply, each ended by a barrier; waves 4..7 run one barrier behind waves 0..3, so
        // that one wave of a SIMD fetches while the other multiplies. A fetch's LDS reads have landed
        // when its barrier opens, so the region they came from is asked for again, for the next use of
        // its stage, in the fetch after that; a fetch waits for what the next one reads, by the number
        // of the wave's younger requests. Up to 14 are under way per wave, 112 KB of the 128 KB of
        // panels. Measured at 8192 x 8192, K 7168: both waves in step 1017 us, turns of 16 MFMAs 727,
        // of 32 664. A third stage of weights in the LDS that is left: 2 % slower. Workgroups that
        // stay and ask for the next tile's first panels before they store: no faster (61 us against
        // 58 for four tiles of one step), as requests wait behind stores.
        u32x4_t wf[2][2][2], xf[4][2];  // [half of the weight rows][tile][columns 32h..], [tile][columns]
        auto read_w = [&](int stage, auto half) __attribute__((always_inline)) {
            const char* wp = ring + stage * STAGE + (wave_n * WN + half * (WN / 2)) * kStepBytes;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    wf[half][i][h] = *reinterpret_cast<const u32x4_t*>(wp + i * 2048 + (frag ^ (h * 64)));
        };
        auto read_x = [&](int stage, auto half) __attribute__((always_inline)) {
            const char* xp = ring + stage * STAGE + (BN + wave_m * WM + half * (WM / 2)) * kStepBytes;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    xf[j][h] = *reinterpret_cast<const u32x4_t*>(xp + j * 2048 + (frag ^ (h * 64)));
        };
        // products of weight half `first` (and, in a whole part, the other half after it) with position half xh
        auto part = [&](auto first, auto both, auto xh) __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            bare_barrier();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int w = 0; w <= both; ++w) {
                const int wh = w == 0 ? first : 1 - first;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[wh * 2 + i][xh * 4 + j] = T::mfma(wf[wh][i][h], xf[j][h], acc[wh * 2 + i][xh * 4 + j]);
            }
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            bare_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        constexpr std::false_type kept{};
        if (t.count > BM / 2) {
            if (full > 0) request(0, 0, C<0>{}, C<8>{}, kept);
            if (full > 1) {
                request(1, 1, C<0>{}, C<6>{}, kept);
                wait_requests<8>();
            } else {
                wait_requests<0>();
            }
            bare_barrier();
            if (wave >= 4) bare_barrier();
            for (int s = 0; s < full; ++s) {
                const int b = s & 1;
                if (s + 1 < full) request(s + 1, b ^ 1, C<6>{}, C<2>{}, kept);
                read_w(b, C<0>{});
                read_x(b, C<0>{});
                read_w(b, C<1>{});
                if (s + 1 < full) wait_requests<8>();  // the second positions of this step
                else wait_requests<0>();
                part(C<0>{}, C<1>{}, C<0>{});
                if (s + 2 < full) request(s + 2, b, C<0>{}, C<6>{}, kept);
                read_x(b, C<1>{});
                if (s + 2 < full) wait_requests<8>();  // the next step's weights and first positions
                else wait_requests<0>();
                part(C<1>{}, C<1>{}, C<1>{});
            }
        } else {
            // no second half of positions: parts of 16 MFMAs, one for each half of the weight rows, and
            // six requests a step, which make it 0.75 of a whole one
            if (full > 0) request(0, 0, C<0>{}, C<6>{}, kept);
            if (full > 1) {
                request(1, 1, C<0>{}, C<4>{}, kept);
                wait_requests<6>();
            } else {
                wait_requests<0>();
            }
            bare_barrier();
            if (wave >= 4) bare_barrier();
            for (int s = 0; s < full; ++s) {
                const int b = s & 1;
                if (s + 1 < full) request(s + 1, b ^ 1, C<4>{}, C<2>{}, kept);
                read_w(b, C<0>{});
                read_x(b, C<0>{});
                if (s + 1 < full) wait_requests<6>();
                else wait_requests<0>();
                part(C<0>{}, C<0>{}, C<0>{});
                if (s + 2 < full) request(s + 2, b, C<0>{}, C<4>{}, kept);
                read_w(b, C<1>{});
                if (s + 2 < full) wait_requests<6>();
                else wait_requests<0>();
                part(C<1>{}, C<0>{}, C<0>{});
            }
        }
        if (wave < 4) bare_barrier();
    } else if constexpr (ALIGNED) {
        // A step's fragments are read while the step before is multiplied; its stage is asked for
        // again, for S steps later, behind the barrier that follows the reads.
        auto ring_loop = [&](auto stream) __attribute__((always_inline)) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (s < full) request(s, s, C<0>{}, C<NI>{}, stream);
            }
            Fragments f[2];
            if (S <= full) wait_requests<(S - 1) * NI>();
            else wait_requests<0>();
            bare_barrier();
            if (full > 0) read_step(f[0], 0);
            int stage = 0;
            auto step = [&](int s, const Fragments& now, Fragments& next) __attribute__((always_inline)) {
                if (s + S - 1 < full) wait_requests<(S - 2) * NI>();  // step s+1 is there, S-2 younger ones are under way
                else wait_requests<0>();
                bare_barrier();
                if (s + S < full) request(s + S, stage, C<0>{}, C<NI>{}, stream);
                stage = stage + 1 == S ? 0 : stage + 1;
                if (s + 1 < full) read_step(next, stage);
                multiply(now);
            };
            for (int s = 0; s < full; s += 2) {
                step(s, f[0], f[1]);
                if (s + 1 < full) step(s + 1, f[1], f[0]);
            }
        };
        if (t.only) ring_loop(std::true_type{});
        else ring_loop(std::false_type{});
    } else {
        // the same through registers: loads two steps ahead of the products, LDS one
        Fragments f[2];
        fetch(0);
        put(0);
        if (steps > 1) fetch(1);
        __syncthreads();
        read_step(f[0], 0);
        if (steps > 1) put(1);
        if (steps > 2) fetch(2);
        auto step = [&](int s, const Fragments& now, Fragments& next) __attribute__((always_inline)) {
            __syncthreads();
            if (s + 1 < steps) read_step(next, (s + 1) & 1);
            multiply(now);
            if (s + 2 < steps) put(s & 1);
            if (s + 3 < steps) fetch(s + 3);
        };
        for (int s = 0; s < steps; s += 2) {
            step(s, f[0], f[1]);
            if (s + 1 < steps) step(s + 1, f[1], f[0]);
        }
    }
    if (ALIGNED && steps > full) {  // the last columns of a K that is no multiple of 64
        Fragments f;
        fetch(full);
        wait_reads();
        bare_barrier();
        put(0);
        wait_reads();
        bare_barrier();
        read_step(f, 0);
        multiply(f);
    }

    // Epilogue. To the matrix instruction lane l is position l%16 and rows 4*(l/16) .. +3 of a 16-row
    // tile. The panel's rows are not in the order of the outputs, though (output_of): two neighbouring
    // tiles give a lane eight outputs in a row and a position's four lanes 32, 64 or 128 bytes, so results
    // go to memory from where they are. (Turned through LDS into whole lines: 7.3 us a 256 x 256 tile.)
    int to[TM];  // row of the output, or draw; -1: nowhere
    float scale[TM];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        const int m = position_of(wave_m * WM + j * 16) + (lane & 15);
        to[j] = m < t.count ? t.first + m : -1;
        if (to[j] >= 0 && a.mode == kProductDraws) {
            const int draw = a.draws[to[j]];
            to[j] = draw >= 0 && draw < a.draw_count ? draw : -1;
            scale[j] = to[j] >= 0 ? a.draw_weights[draw] : 0.0f;
        } else if (to[j] >= 0 && a.rows != nullptr) {
            const int row = a.rows[to[j]];
            if (row < 0 || row >= a.x_rows) to[j] = -1;
        }
    }
    auto finish = [&](auto pair) __attribute__((always_inline)) {
        constexpr int TILES = pair ? TN / 2 : TN;   // of outputs
        constexpr int RUN = TILES >= 2 ? 2 : 1;     // tiles that share a lane's outputs in a row
        constexpr int V = RUN * 4, GROUPS = TILES / RUN;
        const int o0 = n0 + wave_n * TILES * 16 + (lane >> 4) * V;  // outputs of group g: o0 + 32 g .. + V - 1
        if (a.mode == kProductPartial) {
            const size_t share = static_cast<size_t>(blockIdx.y) * (a.pair + 1) * a.positions;
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                if (to[j] < 0) continue;
#pragma unroll
                for (int i = 0; i < TN; ++i) {
                    const int o = o0 + i % TILES / RUN * 32 + i % RUN * 4;
                    store_wide(a.wide + (share + static_cast<size_t>(i / TILES) * a.positions + to[j]) * a.n + o, acc[i][j], o, a.n);
                }
            }
            return;
        }
        float4_t bias[TN];  // the same for every position
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int o = o0 + i % TILES / RUN * 32 + i % RUN * 4;
            const uint16_t* from = a.bias[i / TILES];
            bias[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (from != nullptr && o < a.n) bias[i] = load_narrow<T>(from + static_cast<size_t>(t.expert) * a.n + o, o, a.n);
        }
        if (a.mode == kProductDraws) {
#pragma unroll
            for (int j = 0; j < TM; ++j) {
                if (to[j] < 0) continue;
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const int o = o0 + i / RUN * 32 + i % RUN * 4;
                    store_wide(a.wide + static_cast<size_t>(to[j]) * a.n + o, (acc[i][j] + bias[i]) * scale[j], o, a.n);
                }
            }
            return;
        }
        Narrow<T, V> ahead[GROUPS];  // residuals of the next position, asked for before this one's stores
        auto residuals = [&](int row) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                if (row >= 0) ahead[g].load(a.residual + row * a.residual_stride + o0 + 32 * g, o0 + 32 * g, a.n);
        };
        if (a.residual != nullptr) residuals(to[0]);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            Narrow<T, V> res[GROUPS];
            if (a.residual != nullptr) {
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) res[g] = ahead[g];
                if (j + 1 < TM) residuals(to[(j + 1) % TM]);
            }
            float y[TILES * 4], u[TILES * 4];
#pragma unroll
            for (int k = 0; k < TILES * 4; ++k) {
                y[k] = acc[k / 4][j][k % 4] + bias[k / 4][k % 4];
                u[k] = pair ? acc[(k / 4 + TILES) % TN][j][k % 4] + bias[(k / 4 + TILES) % TN][k % 4] : 0.0f;
            }
            activate(a.activation, y, u, a.limit);
            if (to[j] < 0) continue;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                float v[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    v[k] = y[g * V + k];
                    if (a.residual != nullptr) v[k] += res[g].value(k);
                }
                Narrow<T, V> out;
                out.round(v);
                out.store(a.y + to[j] * a.y_stride + o0 + 32 * g, o0 + 32 * g, a.n);
            }
            __builtin_amdgcn_sched_barrier(0);  // one position at a time: the accumulators fill the registers
        }
    };
    if (a.pair) finish(std::true_type{});
    else finish(std::false_type{});
}

// ---- a few positions: one pass of the weights through registers ------------------------------------
//
// Up to four positions do not fill an MFMA tile, and the latency of a stage ring is most of such a
// call. Here a wave's lanes lie along K (16 bytes each, 512 columns a load), the four waves of a
// workgroup take turns at the 512-column chunks, and every wave keeps R rows' loads in flight with no
// LDS or barrier before the final sum: lanes by butterfly, waves in order. Bound by the weight stream,
// or by launch and one trip to memory where the matrix is small. R = 8 rows of one matrix (4 of each
// where there are two, fewer where the matrix has too few rows for the CUs).

template <class T>
__device__ __forceinline__ void widen8(const u32x4_t& v, float out[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[2 * i] = T::widen(static_cast<uint16_t>(v[i] & 0xFFFFu));
        out[2 * i + 1] = T::widen(static_cast<uint16_t>(v[i] >> 16));
    }
}

// Dots of R weight rows with TOK rows of x over this wave's chunks of K: acc[r][t] += this lane's part.
// Of a last chunk that K cuts, a lane loads the row's last eight values at most and masks those that
// the lane before it has: every load stays inside its row (so K has at least eight columns).
template <class T, int R, int TOK>
__device__ __forceinline__ void row_dots(const uint16_t* const (&w)[R], const uint16_t* const (&x)[TOK], int k, int wave,
                                         int waves, int lane, float (&acc)[R][TOK]) {
    typedef u32x4_t __attribute__((aligned(2))) loose_t;
    auto chunk = [&](int c, auto cut, u32x4_t keep) __attribute__((always_inline)) {
        u32x4_t wv[R];
#pragma unroll
        for (int r = 0; r < R; ++r) wv[r] = __builtin_nontemporal_load(reinterpret_cast<const AEON_GLOBAL loose_t*>(as_global<uint16_t>(w[r]) + c));
        float xv[TOK][8];
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
            u32x4_t v = *reinterpret_cast<const AEON_GLOBAL loose_t*>(as_global<uint16_t>(x[t]) + c);
            if (cut) v &= keep;
            widen8<T>(v, xv[t]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float wf[8];
            if (cut) wv[r] &= keep;
            widen8<T>(wv[r], wf);
#pragma unroll
            for (int t = 0; t < TOK; ++t)
#pragma unroll
                for (int q = 0; q < 8; ++q) acc[r][t] = fmaf(wf[q], xv[t][q], acc[r][t]);
        }
    };
    int at = wave * 512;
    for (; at + 512 <= k; at += waves * 512) chunk(at + lane * 8, std::false_type{}, u32x4_t{});
    if (at < k) {
        const int c = at + lane * 8;
        const int from = c < k - 8 ? c : k - 8;
        u32x4_t keep;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            keep[i] = (from + 2 * i >= c ? 0xFFFFu : 0u) | (from + 2 * i + 1 >= c ? 0xFFFF0000u : 0u);
        chunk(from, std::true_type{}, keep);
    }
}

constexpr int kFewWaves = 4;
constexpr int kFewMax = 4;  // positions of a window
constexpr int kFewColumns = 8;
constexpr int kFewTokens = 16;  // of a dense product that may still be cheapest in a few such windows

template <class T, int ROWS, int MATS, int TOK>
__device__ __forceinline__ void few_body(const ProductArgs& a, const ProductTile& t, float (*sums)[kFewWaves]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = t.row_block * ROWS;
    const uint16_t* w[ROWS * MATS];
#pragma unroll
    for (int r = 0; r < ROWS * MATS; ++r) {
        const int row = n0 + r % ROWS < a.n ? n0 + r % ROWS : a.n - 1;
        w[r] = a.w[r / ROWS] + t.expert * a.expert_stride + row * a.w_stride;
    }
    const uint16_t* x[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
        int m = t.first + (i < t.count ? i : t.count - 1);
        if (a.rows != nullptr) {
            m = a.rows[m];
            m = m < 0 ? 0 : (m < a.x_rows ? m : a.x_rows - 1);
        }
        x[i] = a.x + m * a.x_stride;
    }
    float acc[ROWS * MATS][TOK] = {};
    row_dots<T>(w, x, a.k, wave, kFewWaves, lane, acc);
#pragma unroll
    for (int r = 0; r < ROWS * MATS; ++r)
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const float v = wave_xor_sum(acc[r][i], 63);
            if (lane == 0) sums[r * TOK + i][wave] = v;
        }
    __syncthreads();
    const int i = threadIdx.x / ROWS, r = threadIdx.x % ROWS, o = n0 + r;
    if (i >= t.count || o >= a.n) return;
    auto total = [&](int m) {
        const float* v = sums[(m * ROWS + r) * TOK + i];
        float s = ((v[0] + v[1]) + v[2]) + v[3];
        if (a.bias[m] != nullptr) s += T::widen(a.bias[m][static_cast<size_t>(t.expert) * a.n + o]);
        return s;
    };
    const int p = t.first + i;
    const float g = total(0);
    if (a.mode == kProductDraws) {
        const long draw = a.draws[p];
        if (draw >= 0 && draw < a.draw_count) a.wide[static_cast<size_t>(draw) * a.n + o] = g * a.draw_weights[draw];
        return;
    }
    if (a.mode == kProductPartial) {
        a.wide[static_cast<size_t>(p) * a.n + o] = g;
        return;
    }
    if (a.rows != nullptr) {
        const int row = a.rows[p];
        if (row < 0 || row >= a.x_rows) return;
    }
    float value[1] = {g}, up[1] = {MATS == 2 ? total(1) : 0.0f};
    activate(a.activation, value, up, a.limit);
    float y = value[0];
    if (a.residual != nullptr) y += T::widen(a.residual[p * a.residual_stride + o]);
    a.y[p * a.y_stride + o] = T::round(y);
}

template <class T, int ROWS, int MATS>
__global__ __launch_bounds__(64 * kFewWaves) void product_few_kernel(const ProductArgs a) {
    __shared__ float sums[ROWS * MATS * kFewMax][kFewWaves];
    ProductTile t;
    if (!find_tile<kFewMax, false>(a, (a.n + ROWS - 1) / ROWS, blockIdx.x, &t)) return;
    if (t.count == 1) few_body<T, ROWS, MATS, 1>(a, t, sums);
    else if (t.count == 2) few_body<T, ROWS, MATS, 2>(a, t, sums);
    else few_body<T, ROWS, MATS, 4>(a, t, sums);
}

// Sums over the lanes of eight values a lane: of value lane % 8. Three exchanges halve the values a lane holds (with
// lane ^ 7, ^ 2 and ^ 1, which reach all eight), three steps add what is left over lanes 8, 16 and 32 apart. All of it in
// the vector pipe, seven moves and three steps: a butterfly through LDS for each value is 48 round trips.
template <int CTRL>
__device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float sum_by_row(const float (&v)[8], int lane) {
    constexpr int kXor7 = 0x141, kXor2 = 0x4E, kXor1 = 0xB1, kXor8 = 0x128;  // row_half_mirror, quad_perm twice, row_ror:8
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (lane & 4 ? v[i + 4] : v[i]) + from_lane<kXor7>(lane & 4 ? v[i] : v[i + 4]);
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (lane & 2 ? a[i + 2] : a[i]) + from_lane<kXor2>(lane & 2 ? a[i] : a[i + 2]);
    float c = (lane & 1 ? b[1] : b[0]) + from_lane<kXor1>(lane & 1 ? b[0] : b[1]);
    c += from_lane<kXor8>(c);
    // the rows of 16 lanes of a pair, then the halves of the wave, change places: the two results add up to the sum
    auto joined = [](auto pair) {
        const uint32_t one = pair[0], two = pair[1];
        return __builtin_bit_cast(float, one) + __builtin_bit_cast(float, two);
    };
    uint32_t bits = __builtin_bit_cast(uint32_t, c);
    bits = __builtin_bit_cast(uint32_t, joined(__builtin_amdgcn_permlane16_swap(bits, bits, false, false)));
    return joined(__builtin_amdgcn_permlane32_swap(bits, bits, false, false));
}

// The weighted sum of a token's expert products in one launch: a workgroup walks the slots of its
// token for ROWS outputs, so nothing passes through memory between the products and the sum. Every
// slot streams its expert's rows anew, hence for a few tokens. The slots' chunks of K follow each
// other in one sequence whose next loads are issued before the present ones are used. At most 64
// draws: lane l holds draw l's id, weight and position. The weight meets a slot's whole product, as in two launches: a
// weighed part may be infinite, or NaN beside an infinite weight, where the product is neither. Measured, us of this
// kernel / of two launches, cold rows: 1, 3 and 4 tokens of 8 slots, 2048 -> 7168: 41.1 / 46.0, 118 / 121 and 162 / 157; 8
// tokens of 2 slots, 1024 -> 1024 (34 MB of rows): 9.0 / 12.5; 6 tokens of 6 slots, 512 -> 2048 (75 MB): 18.3 / 20.9. With rows
// that repeat the two launches were ahead from 50 MB on. The host spends 4 us less on it.
constexpr int kDirectDraws = 64;
constexpr int kDirectTokens = 3;
constexpr double kDirectBytes = 40e6;  // rows streamed, above which more tokens go through memory
template <class T, int ROWS>
__global__ __launch_bounds__(64 * kFewWaves) void product_token_kernel(const ProductArgs a, const int32_t* ids, int slots,
                                                                       const uint16_t* base, long base_stride,
                                                                       uint16_t* out, long out_stride) {
    typedef u32x4_t __attribute__((aligned(2))) loose_t;
    __shared__ float sums[kDirectDraws][ROWS][kFewWaves];  // by slot
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token = blockIdx.y;
    const int n0 = blockIdx.x * ROWS;
    int listed = a.offsets[a.experts];
    listed = listed < a.positions ? listed : a.positions;
    const int draw_here = lane < listed ? a.draws[lane] : -1;
    const int own = token * slots + lane;
    const int id = lane < slots ? ids[own] : -1;
    const float weight = lane < slots ? a.draw_weights[own] : 0.0f;
    int position = -1;
    for (int s = 0; s < slots; ++s) {
        const uint64_t at = __ballot(draw_here == token * slots + s);
        if (lane == s && at != 0) position = __builtin_ctzll(at);
    }
    // a slot whose id names no expert, or that no list holds, is left out
    uint64_t slots_left = __ballot(lane < slots && id >= 0 && id < a.experts && position >= 0);

    // the sequence (slot, chunk of 512 columns): this wave's chunks are wave, wave + 4, ...
    int slot = 0, at = a.k;
    auto next = [&]() __attribute__((always_inline)) {  // false when the sequence has ended
        at += kFewWaves * 512;
        if (at < a.k) return true;
        if (wave * 512 >= a.k || slots_left == 0) return false;
        slot = __builtin_ctzll(slots_left);
        slots_left &= slots_left - 1;
        at = wave * 512;
        return true;
    };
    struct Load {
        u32x4_t w[ROWS], x;
        int slot, c;
        bool last;  // of the slot's chunks in this wave
    } load[2];
    auto issue = [&](Load& l) __attribute__((always_inline)) {
        const int expert = __builtin_amdgcn_readlane(id, slot);
        const int p = __builtin_amdgcn_readlane(position, slot);
        const int c = at + lane * 8;
        const int from = c < a.k - 8 ? c : a.k - 8;
        l.slot = slot;
        l.c = c;
        l.last = at + kFewWaves * 512 >= a.k;
        const AEON_GLOBAL uint16_t* w = as_global<uint16_t>(a.w[0]) + expert * a.expert_stride;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int row = n0 + r < a.n ? n0 + r : a.n - 1;
            l.w[r] = __builtin_nontemporal_load(reinterpret_cast<const AEON_GLOBAL loose_t*>(w + row * a.w_stride + from));
        }
        l.x = *reinterpret_cast<const AEON_GLOBAL loose_t*>(as_global<uint16_t>(a.x) + p * a.x_stride + from);
    };
    float dot[ROWS] = {};
    auto use = [&](Load& l) __attribute__((always_inline)) {
        u32x4_t keep;  // the values before column c are the lane before's (row_dots)
        const int over = l.c < a.k - 8 ? 0 : l.c - (a.k - 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = (2 * i >= over ? 0xFFFFu : 0u) | (2 * i + 1 >= over ? 0xFFFF0000u : 0u);
        float x[8];
        widen8<T>(l.x & keep, x);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float w[8];
            widen8<T>(l.w[r] & keep, w);
#pragma unroll
            for (int q = 0; q < 8; ++q) dot[r] = fmaf(w[q], x[q], dot[r]);
        }
        if (!l.last) return;
        const float sum = sum_by_row(dot, lane);
        if (lane < ROWS) sums[l.slot][lane][wave] = sum;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) dot[r] = 0.0f;
    };
    const uint64_t all_slots = slots_left;
    bool more = next();
    if (more) issue(load[0]);
    while (more) {
        const bool second = next();
        if (second) issue(load[1]);
        use(load[0]);
        if (!second) break;
        more = next();
        if (more) issue(load[0]);
        use(load[1]);
    }
    __syncthreads();
    if (wave != 0) return;
    const int waves = (a.k + 511) / 512 < kFewWaves ? (a.k + 511) / 512 : kFewWaves;  // that had a chunk
    const int o = n0 + lane;
    const bool live = lane < ROWS && o < a.n;
    float y = 0.0f;
    if (live && base != nullptr) y = T::widen(base[token * base_stride + o]);
    for (uint64_t left = all_slots; left != 0; left &= left - 1) {
        const int s = __builtin_ctzll(left);
        const float scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), s));
        const int expert = __builtin_amdgcn_readlane(id, s);
        if (live) {
            float v = sums[s][lane][0];
            for (int i = 1; i < waves; ++i) v += sums[s][lane][i];
            if (a.bias[0] != nullptr) v += T::widen(a.bias[0][static_cast<size_t>(expert) * a.n + o]);
            y += v * scale;
        }
    }
    if (live) out[token * out_stride + o] = T::round(y);
}

// Joins the shares of K of a dense product, in share order, and applies the epilogue, or leaves the sums in `sums`
// as they are (a product without epilogue). Four outputs a thread.
template <class T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs a, int splits, float* sums) {
    const int groups = (a.n + 3) / 4;
    const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= static_cast<long>(a.positions) * groups) return;
    const int p = static_cast<int>(at / groups);
    const int o = static_cast<int>(at - static_cast<long>(p) * groups) * 4;
    const int mats = a.pair + 1;
    float4_t sum[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    const size_t share = static_cast<size_t>(a.positions) * a.n;
    for (int s = 0; s < splits; ++s) {
        const float* src = a.wide + static_cast<size_t>(s) * mats * share + static_cast<size_t>(p) * a.n + o;
        sum[0] += load_wide(src, o, a.n);
        if (a.pair) sum[1] += load_wide(src + share, o, a.n);
    }
    if (sums != nullptr) {
        store_wide(sums + static_cast<size_t>(p) * a.n + o, sum[0], o, a.n);
        return;
    }
    float v[4], u[4];
    if (a.bias[0] != nullptr) sum[0] += load_narrow<T>(a.bias[0] + o, o, a.n);
    if (a.bias[1] != nullptr) sum[1] += load_narrow<T>(a.bias[1] + o, o, a.n);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        v[q] = sum[0][q];
        u[q] = sum[1][q];
    }
    activate(a.activation, v, u, a.limit);
    float4_t y = {v[0], v[1], v[2], v[3]};
    if (a.residual != nullptr) y += load_narrow<T>(a.residual + p * a.residual_stride + o, o, a.n);
    store_narrow<T>(a.y + p * a.y_stride + o, y, o, a.n);
}

// out[t][i] = round(base[t][i] + sum of the token's contributions in slot order). A draw whose id
// is outside [0, experts) holds no contribution and is left out. Four outputs a thread, one token a
// workgroup, eight slots' loads in flight.
template <class T>
__global__ __launch_bounds__(256) void product_combine_kernel(const float* __restrict__ contrib,
                                                              const int32_t* __restrict__ ids, int experts,
                                                              int blocks, int slots, int n, const uint16_t* base,
                                                              long base_stride, uint16_t* out, long out_stride) {
    const int t = blockIdx.x / blocks;
    const int o = ((blockIdx.x - t * blocks) * 256 + threadIdx.x) * 4;
    if (o >= n) return;
    const long draw = static_cast<long>(t) * slots;
    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (base != nullptr) sum = load_narrow<T>(base + t * base_stride + o, o, n);
    for (int s = 0; s < slots; s += 8) {
        float4_t v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int id = s + k < slots ? ids[draw + s + k] : -1;
            v[k] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (id >= 0 && id < experts) v[k] = load_wide(contrib + static_cast<size_t>(draw + s + k) * n + o, o, n);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += v[k];
    }
    store_narrow<T>(out + t * out_stride + o, sum, o, n);
}

// ---- launches --------------------------------------------------------------------------------

// Tiles, positions x weight rows. 128 x 128 is there twice: two workgroups of two stages a CU, for
// many tiles, or one of four stages and twice the waves.
enum Tile : int { kTileFew, kTile16x64, kTile32x64, kTile32x32, kTile64x64, kTile64x32, kTile128Pair, kTile128Alone, kTile256 };

// A launch counts its threads in 32 bits.
static int check_grid(long workgroups, int threads) {
    AEON_REQUIRE(workgroups <= 0xffffffffL / threads, AEON_ERR_INVALID_ARGUMENT,
                 "product: %ld workgroups are more than one launch holds", workgroups);
    return AEON_OK;
}

template <class T, int BM, int BN, int WAVES_M, int WAVES_N, int S, bool ALIGNED>
static int launch_tile(const ProductArgs& a, int splits, hipStream_t stream) {
    auto kernel = product_kernel<T, BM, BN, WAVES_M, WAVES_N, S, ALIGNED>;
    constexpr int bytes = S * (BM + BN) * kStepBytes;
    const long rows = a.pair ? BN / 2 : BN;
    const long row_blocks = (a.n + rows - 1) / rows;
    // an upper bound of the windows: every list that holds something may end in a short one
    long windows = (static_cast<long>(a.positions) + BM - 1) / BM;
    if (a.offsets != nullptr) windows = a.positions / BM + (a.experts < a.positions ? a.experts : a.positions);
    long grid = (windows * row_blocks + kXcds - 1) / kXcds * kXcds;
    // room for a last round in halves
    if (takes_turns(BM, ALIGNED) && a.offsets == nullptr) grid += kXcds * (kXcdCus / 2);
    if (int rc = check_grid(grid, 64 * WAVES_M * WAVES_N)) return rc;
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
    kernel<<<dim3(static_cast<unsigned>(grid), splits), 64 * WAVES_M * WAVES_N, bytes, stream>>>(a);
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}

// Rows of each matrix a workgroup of the few-position kernel takes: eight loads in flight a wave, or
// fewer where that would leave CUs without a workgroup (2 a CU at least).
template <class T, int ROWS, int MATS>
static int launch_few_rows(const ProductArgs& a, long windows, hipStream_t stream) {
    const long grid = (windows * ((a.n + ROWS - 1) / ROWS) + kXcds - 1) / kXcds * kXcds;
    if (int rc = check_grid(grid, 64 * kFewWaves)) return rc;
    product_few_kernel<T, ROWS, MATS><<<static_cast<unsigned>(grid), 64 * kFewWaves, 0, stream>>>(a);
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}

template <class T>
static int launch_few(const ProductArgs& a, hipStream_t stream) {
    long windows = (static_cast<long>(a.positions) + kFewMax - 1) / kFewMax;
    if (a.offsets != nullptr) windows = a.positions / kFewMax + (a.experts < a.positions ? a.experts : a.positions);
    const long rows = windows * a.n;
    if (a.pair) return rows >= 4 * 512 ? launch_few_rows<T, 4, 2>(a, windows, stream) : launch_few_rows<T, 1, 2>(a, windows, stream);
    if (rows >= 8 * 512) return launch_few_rows<T, 8, 1>(a, windows, stream);
    return rows >= 4 * 512 ? launch_few_rows<T, 4, 1>(a, windows, stream) : launch_few_rows<T, 1, 1>(a, windows, stream);
}

template <class T, bool ALIGNED>
static int launch_tiles(Tile tile, const ProductArgs& a, int splits, hipStream_t stream) {
    if constexpr (ALIGNED) {
        switch (tile) {
            case kTile16x64: return launch_tile<T, 16, 64, 1, 2, 7, true>(a, splits, stream);
            case kTile32x64: return launch_tile<T, 32, 64, 1, 2, 6, true>(a, splits, stream);
            case kTile32x32: return launch_tile<T, 32, 32, 2, 1, 9, true>(a, splits, stream);
            case kTile64x64: return launch_tile<T, 64, 64, 2, 2, 5, true>(a, splits, stream);
            case kTile64x32: return launch_tile<T, 64, 32, 4, 1, 6, true>(a, splits, stream);
            case kTile128Pair: return launch_tile<T, 128, 128, 2, 2, 2, true>(a, splits, stream);
            case kTile128Alone: return launch_tile<T, 128, 128, 2, 4, 4, true>(a, splits, stream);
            default: return launch_tile<T, 256, 256, 2, 4, 2, true>(a, splits, stream);
        }
    } else {
        switch (tile) {
            case kTile16x64:
            case kTile32x64:
            case kTile32x32: return launch_tile<T, 32, 64, 1, 2, 2, false>(a, splits, stream);
            case kTile64x64:
            case kTile64x32: return launch_tile<T, 64, 64, 2, 2, 2, false>(a, splits, stream);
            default: return launch_tile<T, 128, 128, 2, 2, 2, false>(a, splits, stream);
        }
    }
}

static bool on_boundary(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

static int launch_product(int dtype, Tile tile, ProductArgs& a, int splits, hipStream_t stream) {
    const bool aligned = on_boundary(a.x, 4) && on_boundary(a.w[0], 4) && on_boundary(a.w[1], 4) && a.x_stride % 2 == 0 &&
                         a.w_stride % 2 == 0 && a.expert_stride % 2 == 0;
    if (tile == kTileFew) return dtype == AEON_DTYPE_F16 ? launch_few<F16>(a, stream) : launch_few<BF16>(a, stream);
    if (dtype == AEON_DTYPE_F16) {
        return aligned ? launch_tiles<F16, true>(tile, a, splits, stream) : launch_tiles<F16, false>(tile, a, splits, stream);
    }
    return aligned ? launch_tiles<BF16, true>(tile, a, splits, stream) : launch_tiles<BF16, false>(tile, a, splits, stream);
}

constexpr int kMostPositions = 1 << 30;  // positions and their sums with a tile's are 32-bit numbers

// A tile and the shares K is cut into.
struct ProductPlan {
    Tile tile;
    int splits, split_steps;
};

// What a tile costs, us: a 64-column step of a workgroup that has its CU to itself, of one of two that
// share it (0: it never does), and the rest of a workgroup (launch, first requests, epilogue). Fitted to
// products of 5 to 4096 tokens with matrices of 1024 x 512 to 14336 x 4096, each at every tile of this table and at one
// to eight shares (120 products; the plan made from these figures is within 0.3 % of the best one measured in the
// mean, and 7 % at worst). The figures order the tiles; they are not times: a matrix that comes from HBM at every
// call takes up to 1.6 times its price (128 tokens, 4096 -> 14336: 25.5, measured 40), and the choice can be off
// (200 tokens, 7168 -> 28672: 146 us in the planned two shares, 122 in one).
// Without the tiles of 32 rows and the 128 x 128 one that has its CU alone the same products take 6 % more in
// the mean: 128 tokens, K 2048, N 4096: 12.5 us, 10.7 with 64 x 32; 512 tokens, K = N = 7168: 82, and 69 with 128 x 128.
struct TileCost {
    Tile tile;
    int positions, rows;
    double step_alone, step_shared, fixed;
};
constexpr TileCost kTileCosts[] = {{kTile32x32, 32, 32, 0.12, 0.29, 2.2}, {kTile64x32, 64, 32, 0.12, 0.27, 2.2},
                                   {kTile64x64, 64, 64, 0.19, 0.39, 3.0}, {kTile128Alone, 128, 128, 0.46, 0.0, 8.1},
                                   {kTile256, 256, 256, 1.43, 0.0, 16.0}};

// Each tile of the table priced at 1, 2, 3, 4, 6 and 8 shares: rounds of workgroups, the weights' way from memory
// (at 9.7 TB/s, what the Infinity Cache gives; HBM 6.7), and the second launch that joins shares with its traffic.
// The figures are of the kernels for rows on 4-byte boundaries: rows off them take the tile nearest to the planned
// one that passes through registers, and its shares. The kernel for a few positions pays by eight
// weight rows: what a workgroup costs beside its loads, more with the FMAs of two or four positions. Measured,
// us in it / in the best tile: 1 token, 4096 -> 256: 3.4 / 8.5, 7168 -> 7168: 21.1 / 22.6, 512 -> 32000: 18.8 / 9.2;
// 4 tokens: 4.5 / 8.6, 26.5 / 21.1, 45.6 / 9.3; 8 tokens, 4096 -> 256: 4.7 / 9.0.
static ProductPlan plan_linear(const aeon_projection& w, int tokens) {
    const double n = static_cast<double>(w.out_dim) * (w.activation == AEON_ACT_SWIGLU ? 2 : 1);
    const int steps = (w.in_dim + kStep - 1) / kStep;
    const double stream = (n + tokens) * w.in_dim * 2 / 9.7e6 + 3.6;
    ProductPlan best{kTileFew, 1, steps};
    double best_us = 0.0;
    if (tokens <= kFewTokens && w.in_dim >= kFewColumns) {
        const double each = (tokens == 1 ? 2.5e-3 : tokens == 2 ? 4.7e-3 : 8.5e-3) + 1.65e-6 * w.in_dim;
        best_us = 1.4 + n / 8 * ((tokens + kFewMax - 1) / kFewMax) * each;
    }
    for (const TileCost& t : kTileCosts) {
        // tiles that would stay half empty, or be far too many. A window of at most 128 positions makes a 256 x 256
        // step no shorter where the weights come from memory. Measured, us in it / in 128 x 128, 128 tokens: 4096 -> 14336:
        // 68 / 46, 7168 -> 28672: 128 / 87; 7168 -> 65536 is the exception, 178 / 193.
        if (t.positions > 64 ? t.positions >= 2L * tokens : t.rows < 64 && (t.positions < 64 ? tokens > 128 : tokens > 512)) continue;
        const double tiles = static_cast<double>((tokens + t.positions - 1) / t.positions) *
                             ((static_cast<long>(n) + t.rows - 1) / t.rows);
        for (int splits : {1, 2, 3, 4, 6, 8}) {
            if (splits > 1 && (splits > steps / 2 || tiles * splits > 1100)) break;
            const int each = (steps + splits - 1) / splits;
            const long groups = static_cast<long>(tiles * splits);
            const int round = t.step_shared > 0.0 ? 512 : 256;
            const long last = groups % round;
            double us = groups / round * (each * (t.step_shared > 0.0 ? t.step_shared : t.step_alone) + t.fixed);
            if (last > 0) {
                double step = last <= 256 ? t.step_alone : t.step_shared;
                // a last round of the waves that take turns is cut into halves of 0.55 of a tile's products
                if (t.tile == kTile256 && last <= 128 && splits == 1) step *= 0.55;
                us += each * step + t.fixed;
            }
            if (us < stream) us = stream;
            if (splits > 1) us += 0.7 + 8.0 * splits * tokens * n / 14.5e6;
            if (best_us == 0.0 || us < best_us) {
                best_us = us;
                best = ProductPlan{t.tile, splits, each};
            }
        }
    }
    best.splits = (steps + best.split_steps - 1) / best.split_steps;
    return best;
}

// Lists. A few positions with small matrices: the kernel that has no ring. Measured, us in it / in 16 x 64 tiles:
// 4 draws over 8 experts of 1024 x 1024: 7.0 / 8.0, 8 draws 13.5 / 8.2; 2 draws of 4096 x 4096: 15.8 / 19.3, 4 draws:
// 28.0 / 28.7; 4 draws of 4096 x 1024: 14.9 / 9.2; 16 draws over 256 of 256 x 1024: 7.8 / 8.7, over 8 of 256 x 128
// (two or three positions an expert): 9.8 / 7; 8 gated draws of 2048 x 7168: 76 / 73.
// Otherwise by how many positions an expert holds on average, and only as large a tile as leaves the CUs
// enough of them (half a window an expert is taken to be short). Measured, us per product at a mean of 16 /
// 32 / 64 / 96 / 128 / 192 positions, 64 experts of 4096 x 2048: tile 32: 172 / 222 / 316 / 407 / 498 / 689;
// 64: 168 / 189 / 262 / 306 / 361 / 489; 128: 185 / 202 / 221 / 240 / 288 / 356; 256: 204 / 207 / 214 / 219 /
// 234 / 273. Gated, 2048 outputs of 4096 columns, at 64 / 96 / 128: 128: 385 / 403 / 528, 256: 408 / 405 /
// 428. Eight experts of 4096 x 4096, tile 64 / 128 / 256, at 96: 66 / 72 / 66; at 192: 106 / 76 / 87; at 256:
// 146 / 131 / 92; tile 32 / 64 at 24: 57 / 49. Tiles of 32 rows, 8 positions in 64 of 4096 x 2048: 190 to 216.
static Tile plan_experts(const aeon_projection& w, int positions, int experts) {
    const int live = experts < positions ? experts : positions;
    const int mean = positions / (live > 0 ? live : 1);
    const long n = static_cast<long>(w.out_dim) * (w.activation == AEON_ACT_SWIGLU ? 2 : 1);
    const bool spread = 2L * positions <= experts;  // mostly one position an expert
    if ((positions <= 4 ? live * n <= 8192 : spread && live * n <= 6144) && w.in_dim >= kFewColumns) return kTileFew;
    auto tiles = [&](long tile) { return (positions / tile + (live + 1) / 2) * ((n + tile - 1) / tile); };
    if (mean > 80 && tiles(256) >= 192) return kTile256;
    if (mean > 48 && tiles(128) >= 400) return kTile128Pair;
    return mean <= 12 ? kTile16x64 : mean <= 20 ? kTile32x64 : kTile64x64;
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
    AEON_REQUIRE(positions >= 0 && positions <= kMostPositions, AEON_ERR_INVALID_ARGUMENT, "%s: position count out of range (%d)",
                 who, positions);
    AEON_REQUIRE(expert_stride >= (w.out_dim - 1) * w.weight_stride + w.in_dim, AEON_ERR_INVALID_ARGUMENT,
                 "%s: expert matrices %ld elements apart overlap", who, expert_stride);
    return AEON_OK;
}

static bool combine_direct(const aeon_projection& w, int tokens, int slots) {
    const long draws = static_cast<long>(tokens) * slots;
    return draws <= kDirectDraws && w.in_dim >= kFewColumns &&
           (tokens <= kDirectTokens || 2.0 * draws * w.in_dim * w.out_dim <= kDirectBytes);
}

static int check_workspace(const void* d_workspace, size_t bytes, size_t need, const char* who) {
    AEON_REQUIRE(bytes >= need && (need == 0 || (d_workspace != nullptr && on_boundary(d_workspace, 16))),
                 AEON_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %zu bytes on a 16-byte boundary (%zu given)", who, need,
                 bytes);
    return AEON_OK;
}

static size_t linear_workspace(const aeon_projection& w, int tokens, const ProductPlan& p) {
    if (p.splits == 1) return 0;
    return static_cast<size_t>(p.splits) * (w.activation == AEON_ACT_SWIGLU ? 2 : 1) * tokens * w.out_dim * sizeof(float);
}

// Shares of K into a.wide, and the launch that joins more than one of them: by the epilogue, or into `sums`.
static int launch_shares(int dtype, const ProductPlan& plan, ProductArgs& a, float* sums, hipStream_t stream) {
    a.mode = kProductPartial;
    a.split_steps = plan.split_steps;
    if (int rc = launch_product(dtype, plan.tile, a, plan.splits, stream)) return rc;
    if (plan.splits == 1) return AEON_OK;
    const long threads = static_cast<long>(a.positions) * ((a.n + 3) / 4);
    const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
    if (dtype == AEON_DTYPE_F16) product_join_kernel<F16><<<blocks, 256, 0, stream>>>(a, plan.splits, sums);
    else product_join_kernel<BF16><<<blocks, 256, 0, stream>>>(a, plan.splits, sums);
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}

}  // namespace aeon355

using namespace aeon355;

extern "C" size_t aeon_linear_workspace_bytes(const aeon_projection* projection, int tokens) {
    if (check_projection(projection, "aeon_linear_workspace_bytes") != AEON_OK || tokens <= 0 || tokens > kMostPositions) return 0;
    return linear_workspace(*projection, tokens, plan_linear(*projection, tokens));
}

extern "C" int aeon_linear(const aeon_projection* projection, const void* d_x, long x_stride, int tokens,
                           const void* d_residual, long residual_stride, void* d_y, long y_stride,
                           void* d_workspace, size_t workspace_bytes, void* stream) {
    const char* who = "aeon_linear";
    if (int rc = check_projection(projection, who)) return rc;
    const aeon_projection& w = *projection;
    AEON_REQUIRE(tokens >= 0 && tokens <= kMostPositions, AEON_ERR_INVALID_ARGUMENT, "%s: token count out of range (%d)", who, tokens);
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
    if (int rc = check_workspace(d_workspace, workspace_bytes, need, who)) return rc;
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
    a.wide = static_cast<float*>(d_workspace);
    return launch_shares(w.dtype, plan, a, nullptr, as_stream(stream));
}

// The gate as a projection without bias or activation.
static aeon_projection gate_projection(const void* d_gate, long gate_stride, int hidden, int experts) {
    return aeon_projection{AEON_DTYPE_BF16, hidden, experts, AEON_ACT_NONE, d_gate, nullptr, gate_stride, nullptr, nullptr, 0.0f};
}

extern "C" size_t aeon_router_logits_bf16_workspace_bytes(int tokens, int hidden, int experts) {
    if (tokens <= 0 || tokens > kMostPositions || hidden <= 0 || experts <= 0) return 0;
    const aeon_projection w = gate_projection(nullptr, hidden, hidden, experts);
    return linear_workspace(w, tokens, plan_linear(w, tokens));
}

extern "C" int aeon_router_logits_bf16(const void* d_x, long x_stride, const void* d_gate_weight, long gate_stride, float* d_logits,
                                       int tokens, int hidden, int experts, void* d_workspace, size_t workspace_bytes,
                                       void* stream) {
    const char* who = "aeon_router_logits_bf16";
    const aeon_projection w = gate_projection(d_gate_weight, gate_stride, hidden, experts);
    if (int rc = check_projection(&w, who)) return rc;
    AEON_REQUIRE(tokens >= 0 && tokens <= kMostPositions, AEON_ERR_INVALID_ARGUMENT, "%s: token count out of range (%d)", who, tokens);
    if (tokens == 0) return AEON_OK;
    AEON_REQUIRE(d_x && d_logits, AEON_ERR_INVALID_ARGUMENT, "%s: null buffer", who);
    AEON_REQUIRE(on_boundary(d_x, 2) && on_boundary(d_logits, 4), AEON_ERR_INVALID_ARGUMENT,
                 "%s: an operand starts off its element's boundary", who);
    AEON_REQUIRE(x_stride >= hidden, AEON_ERR_INVALID_ARGUMENT, "%s: bad row pitch (x %ld)", who, x_stride);
    AEON_REQUIRE(d_logits != d_x && d_logits != d_gate_weight, AEON_ERR_INVALID_ARGUMENT,
                 "%s: the output must not alias the activations or the weights", who);
    const ProductPlan plan = plan_linear(w, tokens);
    if (int rc = check_workspace(d_workspace, workspace_bytes, linear_workspace(w, tokens, plan), who)) return rc;
    ProductArgs a = projection_args(w);
    a.x = static_cast<const uint16_t*>(d_x);
    a.x_stride = x_stride;
    a.x_rows = tokens;
    a.positions = tokens;
    // one share of K is the whole sum: it goes where a share would
    a.wide = plan.splits == 1 ? d_logits : static_cast<float*>(d_workspace);
    return launch_shares(w.dtype, plan, a, d_logits, as_stream(stream));
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
    return launch_product(w.dtype, plan_experts(w, positions, experts), a, 1, as_stream(stream));
}

extern "C" size_t aeon_expert_combine_workspace_bytes(const aeon_projection* projection, int tokens, int slots) {
    if (check_projection(projection, "aeon_expert_combine_workspace_bytes") != AEON_OK || tokens <= 0 || slots <= 0 ||
        static_cast<long>(tokens) * slots > kMostPositions || combine_direct(*projection, tokens, slots))
        return 0;
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
    AEON_REQUIRE(tokens >= 0 && slots > 0 && static_cast<long>(tokens) * slots <= kMostPositions, AEON_ERR_INVALID_ARGUMENT,
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
    if (int rc = check_workspace(d_workspace, workspace_bytes, need, who)) return rc;
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
    const auto* base = static_cast<const uint16_t*>(d_base);
    auto* out = static_cast<uint16_t*>(d_out);
    if (combine_direct(w, tokens, slots)) {
        const dim3 grid((w.out_dim + 7) / 8, tokens);
        if (w.dtype == AEON_DTYPE_F16)
            product_token_kernel<F16, 8><<<grid, 64 * kFewWaves, 0, as_stream(stream)>>>(a, d_topk_ids, slots, base, base_stride, out, out_stride);
        else
            product_token_kernel<BF16, 8><<<grid, 64 * kFewWaves, 0, as_stream(stream)>>>(a, d_topk_ids, slots, base, base_stride, out, out_stride);
        AEON_LAUNCH_CHECK();
        return AEON_OK;
    }
    const int row_blocks = (w.out_dim + 1023) / 1024;
    const long blocks = static_cast<long>(tokens) * row_blocks;
    if (int rc = check_grid(blocks, 256)) return rc;
    if (int rc = launch_product(w.dtype, plan_experts(w, a.positions, experts), a, 1, as_stream(stream))) return rc;
    const auto grid = static_cast<unsigned>(blocks);
    if (w.dtype == AEON_DTYPE_F16) {
        product_combine_kernel<F16><<<grid, 256, 0, as_stream(stream)>>>(a.wide, d_topk_ids, experts, row_blocks, slots, w.out_dim,
                                                                        base, base_stride, out, out_stride);
    } else {
        product_combine_kernel<BF16><<<grid, 256, 0, as_stream(stream)>>>(a.wide, d_topk_ids, experts, row_blocks, slots, w.out_dim,
                                                                         base, base_stride, out, out_stride);
    }
    AEON_LAUNCH_CHECK();
    return AEON_OK;
}
