// attn_paged.cu — attention over a paged key-value cache: one new token per sequence, or the tokens of a
// prompt chunk with a sliding window and first rows that stay visible.
//
// Mathematics: o_h = sum_j exp(s_hj - lse_h) k_j with s_hj = scale q_h . k_j over the visible rows j and
// lse_h = log(sum_j exp(s_hj) + exp(sink_h)).  One row is key and value of every head (the reference's
// cache has one KV head; cuda/flash_attn.cu:148-313).
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "device_utils.cuh"
#include "kernels.cuh"
#include "tcgen05_utils.cuh"

namespace ds4b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------------------------- tensor cores
//
// An item is up to 64 query rows that share their cache rows: the heads of one token (of up to 64 / n_heads tokens, when a chunk's
// heads are few).  A CTA walks over tiles of 64 cache rows, with a role for each of its 20 warps:
//   * eight load the tile's rows, turn them into f16 and store them once, as 128-byte rows of 64 dims with the 128-byte
//     swizzle.  The same bytes serve both products: as the K-major B operand of S = Q K^T and as the M-contiguous A
//     operand of O^T += V^T P^T, since a key row is its value row;
//   * one issues S (M 64 query rows, N 64 cache rows, K head_dim), one, per 128 dims of the output, O^T (M 128 dims, N 64 query rows,
//     K 64 cache rows).  O^T takes 64 tensor-memory columns per 128 dims, so 512 dims and two S buffers fit; O itself (64
//     rows, 512 columns) would leave no room for S.  S of tile n + 1 is issued ahead of O^T of tile n, so the tensor
//     cores work while the softmax of a tile runs;
//   * eight take S from tensor memory, keep the running maximum and sum of the softmax in f32, and leave the weights as f16 (half a
//     step: 2^-11 of each; see kLift) in shared memory.  The accumulators are rescaled only when a row's maximum has grown by more
//     than 2^8 since its last reference, which later tiles rarely bring;
//   * one hands out the items, one looks the tiles' rows up in the page table and touches them ahead of the loads.
//
// Scales.  A cache row is a row factor times f16 numbers.  Rows of ordinary size have the factor 1: codes times a scale that is a power
// of two are exact in f16 where the product is a multiple of 2^-24 (a scale of 2^-15 and above; below, and in blocks far smaller than their
// row's largest, a value is off by up to 2^-25 of the factor), codes times another scale are rounded (scale and product, 2^-11 each), as
// f32 rows and tails are (2^-11).  A row whose scale or tail is far from one keeps a factor r_j, which enters the scores, and as
// log2 r_j the exponent of the weights, so that P holds r_j exp(s_j - M) (times kLift, and below 2^15) and the sum takes P / r_j back.  A query row whose
// largest value is outside [2^-4, 2^15] is scaled by a power of two: bf16's 8 bits fit f16, but for values below
// 2^-17, which are off by up to 2^-25.
//
// Work.  Where items are long and few the list of all tiles is cut into equal runs, one per CTA; an item that several CTAs share
// leaves partial sums (f32 O^T, M and l) that attn_join_kernel adds in order.  Else each CTA takes whole items.  Of a chunk the rows
// may be packed as f16 once (attn_pack_kernel); a tile is then eight TMA boxes, and the loaders fetch query rows and drain
// O^T instead, beside the softmax of the next item.
//
// Bound.  Shared memory: a tile of 512 dims is 64 KiB written and, by the MMAs, 224 KiB read at 128 bytes a cycle, 2300 cycles with nothing
// else on the port (an MMA of M 64, N 64, K 16 reads 4 KiB in 32); the loads' own pass through L1, the weights and the query rows come on
// top.  Measured, as the slope over 8 to 48 tiles a CTA of one session (64 heads): 1.7 us a tile of FP8 rows (3400 cycles at 1965 MHz),
// 2.2 of codes with a tail, 4.2 of f32 rows; start, partial sums and join take 18 to 21 us besides.  From HBM a tile of FP8 rows
// needs 1400 cycles, of f32 rows 5600.  Halves of the MMAs' traffic would need the codes themselves as operands, and the weights as two
// or three 8-bit pieces.  Whole calls: one session of 131072 rows, codes with a tail: 55 us (96 MB, 1.7 TB/s); 64 sequences of up to 16384
// FP8 rows: 90 us (162 MB, 1.8 TB/s; tensor pipe 33 %); 96 sequences, 16 heads, f32 rows, window 1024: 61 us (158 MB, 2.6 TB/s); 4096
// chunk tokens, window 128 + 4 first rows: 176 to 187 us (538 MB, 2.9 to 3.1 TB/s; tensor pipe 31 %), a chain of S, softmax, product and
// drain per token.
constexpr int kCtas = 148;
constexpr int kRows = 64;                   // query rows of an item, cache rows of a tile
constexpr int kSoftWarps = 8, kLoadWarp0 = 8, kLoadWarps = 8, kMmaWarp = 16;
constexpr int kThreads = 20 * 32;
// Registers a thread by role, out of what the block is launched with: a larger sum would wait for registers for ever.
constexpr int kLaunchRegs = 96, kSoftRegs = 72, kLoadRegs = 136, kOtherRegs = 56;
static_assert(kSoftWarps * kSoftRegs + kLoadWarps * kLoadRegs + (20 - kSoftWarps - kLoadWarps) * kOtherRegs <= 20 * kLaunchRegs, "register split");
constexpr int kSplitItems = 4 * kCtas;      // more of them are not cut, see launch_fmt()
constexpr int kWholeTiles = 3;              // items of up to so many tiles are not cut
constexpr int kMinTiles = 2;                // of a run: below, the join costs more than the run saves
constexpr float kRescale = 8.0f;            // log2 units
constexpr float kLift = 0x1p7f;              // of the weights as stored, and so of the accumulators
constexpr int kScaleSets = 4;
constexpr float kLeast = 0x1p-100f;         // of a row's factor
constexpr uint32_t kTmem = 0;               // all 512 columns are allocated, so they begin at column 0

struct Meta { int64_t row0; int rows, h0, parts, pad; };

constexpr int kPacked = 3;                  // in place of a row format: the call's rows lie packed as f16, see attn_pack_kernel

// Where the rows that sequence b's tokens see lie when packed: its first `first` rows, then rows lo .. len - 1, then 16 rows of zeros.
struct Packed {
    int len, lo, first;
    int64_t off;
};
__host__ __device__ constexpr int64_t packed_gap(int window, int n_first, int64_t all_rows) {
    return window > 0 ? (int64_t)window - 1 + n_first + 16 : all_rows + 16;
}
// Tokens [x, y) of sequence b: within [0, n_tokens] whatever q_start holds, so that no index leaves its buffer.
__device__ __forceinline__ int first_token(const AttnArgs &a, int b) { return min(max(a.q_start[b], 0), (int)a.n_tokens); }
__device__ __forceinline__ int2 tokens_of(const AttnArgs &a, int b) {
    const int q0 = first_token(a, b);
    return make_int2(q0, max(first_token(a, b + 1), q0));
}
__device__ __forceinline__ Packed get_packed(const AttnArgs &a, int b) {
    const int64_t most = a.table_width * a.kv.page_rows;
    Packed k;
    const int2 q = tokens_of(a, b);
    k.len = (int)min((int64_t)max(a.kv_len[b], 0), most);
    const int p0 = k.len - (q.y - q.x);
    k.lo = a.window > 0 && p0 + 1 > a.window ? p0 + 1 - a.window : 0;
    k.first = min(a.n_first, k.lo);
    k.off = b * packed_gap(a.window, a.n_first, most) + (a.window > 0 ? max(q.x - first_token(a, 0), 0) : 0);
    return k;
}

// The rows an item sees are a list of two runs, each in tiles of 64: `na` rows, then n - na.  Straight from the cache it is one run: the
// `first` first rows of the sequence, then row lo on.  Packed, rows lo .. come first and the first rows are a run of their own,
// so that every tile is one box of neighbouring rows.
struct Item {
    int64_t row0;                           // first row of q / out, n_heads rows per token
    int b, rows, h0, p0, first, lo, n, na, tiles;
    int at_a, at_b;                         // packed rows where the runs begin
};
__device__ __forceinline__ int first_run_tiles(const Item &it) { return (it.na + 63) >> 6; }
__device__ __forceinline__ int rows_in_tile(const Item &it, int t) {
    const int ta = first_run_tiles(it);
    return min(64, t < ta ? it.na - 64 * t : it.n - it.na - 64 * (t - ta));
}

template <bool PACKED>
__device__ __forceinline__ Item get_item(const AttnArgs &a, int group, int head_groups, int slot) {
    Item it;
    const int g = slot / head_groups, hg = slot - g * head_groups;
    int tok0, ntok = 1;
    if (a.q_start) {
        // sequence b's groups take the slots from q_start[b] / group + b on (one slot per sequence may stay empty)
        int lo = 0, hi = a.n_seqs - 1;
        const int off = first_token(a, 0) / group;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first_token(a, mid) / group + mid - off <= g) lo = mid; else hi = mid - 1;
        }
        it.b = lo;
        const int2 q = tokens_of(a, lo);
        const int local = (g - (q.x / group + lo - off)) * group;
        tok0 = q.x + local;
        ntok = local < 0 ? 0 : min(group, q.y - tok0);
        it.p0 = local - (q.y - q.x);
    } else {
        it.b = tok0 = g;
        it.p0 = -1;
    }
    const int64_t most = a.table_width * a.kv.page_rows;
    it.p0 += (int)min((int64_t)max(a.kv_len[it.b], 0), most);
    const int last = it.p0 + ntok - 1;
    it.lo = a.window > 0 && it.p0 + 1 > a.window ? it.p0 + 1 - a.window : 0;
    it.first = min(a.n_first, it.lo);
    it.n = max(0, it.first + last + 1 - it.lo);
    it.na = it.n;
    it.at_a = it.at_b = 0;
    if (PACKED) {
        const Packed k = get_packed(a, it.b);
        it.na = max(0, it.n - it.first);
        it.at_a = (int)(k.off + k.first + it.lo - k.lo);
        it.at_b = (int)k.off;
    }
    it.tiles = ntok <= 0 ? 0 : max(1, ((it.na + 63) >> 6) + ((it.n - it.na + 63) >> 6));
    it.row0 = (int64_t)tok0 * a.n_heads + hg * kRows;
    it.h0 = hg * kRows;
    it.rows = head_groups > 1 ? min(kRows, a.n_heads - hg * kRows) : ntok * a.n_heads;
    return it;
}

__device__ __forceinline__ long long block_scan64(long long v, long long *scratch, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) { const long long t = scratch[w]; before += w < warp ? t : 0; all += t; }
    __syncthreads();
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ void e4m3x4(uint32_t four, uint32_t &lo, uint32_t &hi) {      // E4M3 -> f16 is exact
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ uint32_t h2b(float x, float y) {         // bf16 pair
    __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t *>(&b);
}
__device__ __forceinline__ uint32_t sat_h2(float x, float y) {      // finite values beyond f16 become +-65504
    x = fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
    y = fabsf(y) < INFINITY ? fminf(fmaxf(y, -65504.f), 65504.f) : y;
    return h2_bits(__floats2half2_rn(x, y));
}
__device__ __forceinline__ uint32_t max_bf16x8(uint4 x, uint32_t m) {      // of the magnitudes, in two halves
    constexpr uint32_t k = 0x7fff7fffu;
    return __vimax3_s16x2(x.w & k, __vimax3_s16x2(x.y & k, x.z & k, x.x & k), m);
}
__device__ __forceinline__ void scale_bf16x8(uint4 &x, float f) {          // f a power of two: exact
    const __nv_bfloat162 m = __float2bfloat162_rn(f);
    uint32_t *y = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<__nv_bfloat162 *>(&y[i]) = __hmul2(*reinterpret_cast<__nv_bfloat162 *>(&y[i]), m);
}
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t x) {
    return h2_bits(__floats2half2_rn(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)));
}
// f16 pairs: infinities and NaN become zeros; whether there were any
template <int N>
__device__ __forceinline__ bool drop_nonfinite(uint32_t (&o)[N]) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t bad = __vcmpeq2(o[i] & 0x7c007c00u, 0x7c007c00u);
        any |= bad;
        o[i] &= ~bad;
    }
    return any != 0;
}
// 2^e and 2^-e with e the exponent of x (0 for x = 0), both normal
__device__ __forceinline__ void pow2_parts(float x, float &up, float &down) {
    int e = (int)((__float_as_uint(x) >> 23) & 255u) - 127;
    if (x == 0.0f) e = 0;
    e = min(max(e, -126), 126);
    up = __uint_as_float((uint32_t)(e + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - e) << 23);
}

// A sink in log2 units, held within f32: beyond that it is heavier, or lighter, than every row all the same.  NaN stays.
__device__ __forceinline__ float sink_log2(float sink) {
    constexpr float most = 3.402823466e38f;
    const float x = sink * kLog2e;
    return x == x ? fminf(fmaxf(x, -most), most) : x;
}

// What the scheduling warp hands to the others: an item and the tiles [t0, t1) of it that this CTA takes; t1 < 0 ends.
struct Segment {
    Item it;
    int t0, t1;
};
constexpr int kSegRing = 4;                 // with the query rows prefetched that far ahead: 8 items ahead 198 us for 4096 tokens, 16 206, 4 179
constexpr int kTileRing = 8;                // tiles the finding warp may be ahead of the loaders
constexpr int kHole = -2;                   // a row without a page
constexpr int kSegReaders = kSoftWarps + 3;  // and the loaders with packed rows
constexpr int kPackCtas = 4 * kCtas, kPackWarps = 8;

struct alignas(64) TcArgs {
    CUtensorMap rows, few;                  // packed f16 rows [packed rows][head_dim], boxes of 64 rows x 64 dims, and of 16 rows
    const float *fac;                       // a factor for each (0: a hole, NaN: a value that is not finite)
    const int *odd;                         // kPackCtas: whether a CTA of the packing has met a factor other than 1
    AttnArgs a;
    int group, head_groups, n_slots, split, page_shift;
    Meta *meta;
    float2 *part_ml;
    float *part_o;
    int *status;
};

__device__ __forceinline__ uint4 ld_row16(const void *p) {          // read once per CTA: no place in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// A row on its way to L2: one instruction of the copy engine, where a prefetch of every line takes the load pipe a cycle each.  p on 16
// bytes, n a multiple of 16.
__device__ __forceinline__ void prefetch_l2(const void *p, int n) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(n) : "memory");
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

struct Bars {
    uint64_t full[2][2], s_full[2], s_free[2], p_full[2], pv_done[2][2], scaled[2], q_full, q_free, o_ready[kScaleSets], o_half, o_done[2], o_free[2], quiet[2];
    uint64_t seg_full[kSegRing], seg_free[kSegRing], tile_full[kTileRing], tile_free[kTileRing];
};

template <int NB, int FMT, bool SHARED>     // NB: head_dim / 128; SHARED: an item may hold several tokens (with packed rows always so)
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ TcArgs g) {
    constexpr int D = NB * 128, kChunks = NB * 2, kTileBytes = kRows * D * 2;
    constexpr int kParts = NB > 2 ? 2 : 1, kPart0 = 2;                 // a tile is handed over in parts: its first 256 dims, the rest
    constexpr bool kPre = FMT == kPacked;
    // Tensor memory: six blocks of 64 columns for O^T, two for S.  With packed rows the items go round the six blocks, so that the
    // products of the next item begin while the last one's accumulators are read: with 512 dims its first two blocks are free
    // at once, the others when two have been read.
    constexpr int kOBlocks = 6, kFree = kOBlocks - NB;
    constexpr uint32_t o_tmem = kTmem, s_tmem = kTmem + kOBlocks * 64;
    auto o_block = [](int base, int b) -> uint32_t { return o_tmem + (uint32_t)(base + b >= kOBlocks ? base + b - kOBlocks : base + b) * 64; };
    auto next_base = [](int base) { return !kPre ? 0 : base + NB >= kOBlocks ? base + NB - kOBlocks : base + NB; };
    const AttnArgs &a = g.a;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *q_s = smem, *k_s = smem + kTileBytes, *p_s = smem + 3 * kTileBytes;
    __shared__ __align__(8) Bars bars_s;
    __shared__ Segment seg_s[kSegRing];
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s, start_slot, start_tile;
    __shared__ long long scan_s[kThreads / 32];
    __shared__ __align__(16) float row_fma[2][2 * kRows], row_div[2][kRows];      // by pairs of rows: factor, factor, addend, addend
    __shared__ __align__(16) int row_at[kPre || !SHARED ? 1 : 2 * kTileRing][kRows];       // a row's place in its sequence
    __shared__ __align__(16) int slot_s[kPre ? 1 : kTileRing][kRows];          // a tile's rows in the pool (-1 past the rows, or kHole), see find_index()
    __shared__ int tile_rows[kTileRing];                            // query rows where a tile is its segment's first, else 0; -1 ends
    __shared__ int64_t tile_row0[kTileRing];                        // and the first of them
    __shared__ float q_mul[kScaleSets][kRows];
    __shared__ __align__(16) float fac_s[2][kRows], inv_s[kScaleSets][kRows];
    __shared__ int odd_s[2], odd_w[2][kLoadWarps];  // 1 + the last tile with a row that is not a plain f16 row: of any loader, of each
    __shared__ int grown_s[2];                      // 1 + the last tile with a row that has grown
    __shared__ int go_s[2][2];                      // see next_segment_together()
    volatile int *abort_flag = &abort_s;
    const uint32_t bars = tc::held(smem_addr(&bars_s));
#define DS4B200_BAR(name, i) (bars + (uint32_t)offsetof(Bars, name) + 8u * (uint32_t)(i))
    int *status = g.status;
    const bool several = SHARED && g.group > 1;         // tokens in an item
    launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

    if (tid == 0) {
        abort_s = 0;
        start_slot = g.n_slots;
        start_tile = 0;
        for (int i = 0; i < 2; ++i) {
            grown_s[i] = odd_s[i] = 0;
            mbar_init(&bars_s.quiet[i], 1); mbar_init(&bars_s.o_done[i], 1); mbar_init(&bars_s.o_free[i], kLoadWarps);
            for (int k = 0; k < kLoadWarps; ++k) odd_w[i][k] = 0;
            mbar_init(&bars_s.scaled[i], kSoftWarps);
            mbar_init(&bars_s.s_full[i], 1); mbar_init(&bars_s.s_free[i], kSoftWarps); mbar_init(&bars_s.p_full[i], kSoftWarps);
            for (int k = 0; k < kParts; ++k) { mbar_init(&bars_s.full[i][k], kPre ? 1 : kLoadWarps); mbar_init(&bars_s.pv_done[i][k], 1); }
        }
        mbar_init(&bars_s.q_full, kLoadWarps); mbar_init(&bars_s.q_free, 1);
        mbar_init(&bars_s.o_half, kLoadWarps);
        // four items: the softmax may be that far ahead of the drain before a product has to wait for it
        for (int i = 0; i < kScaleSets; ++i) mbar_init(&bars_s.o_ready[i], kSoftWarps);
        for (int i = 0; i < kTileRing; ++i) { mbar_init(&bars_s.tile_full[i], 1); mbar_init(&bars_s.tile_free[i], kLoadWarps); }
        for (int i = 0; i < kSegRing; ++i) { mbar_init(&bars_s.seg_full[i], 1); mbar_init(&bars_s.seg_free[i], kSegReaders + (kPre ? kLoadWarps : 0)); }
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // This CTA's share of the tiles: with `split` a run of the list of all of them, else whole items, every gridDim.x-th.
    long long per = 1, left = 1ll << 62;
    if (!kPre && g.split) {
        __syncthreads();
        // every thread has the items tid, tid + kThreads, ..: their tiles are counted once, then the run's first one is found
        constexpr int kMine = (kSplitItems + kThreads - 1) / kThreads;
        int tiles[kMine];
        long long before[kMine], total = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int s = i * kThreads + tid;
            tiles[i] = 0;
            before[i] = total;
            if (i * kThreads >= g.n_slots) continue;
            if (s < g.n_slots) tiles[i] = get_item<kPre>(a, g.group, g.head_groups, s).tiles;
            long long sum;
            before[i] += block_scan64(tiles[i], scan_s, &sum);
            total += sum;
        }
        per = max((long long)kMinTiles, (total + kCtas - 1) / kCtas);
        const long long from = per * blockIdx.x;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (before[i] <= from && from < before[i] + tiles[i]) { start_slot = i * kThreads + tid; start_tile = (int)(from - before[i]); }
        left = min(per, total - per * (long long)blockIdx.x);
    }
    tc::fence_before();
    bool any_factor = false;                             // packed rows: there are factors to look at
    if (kPre) {
        wait_dependency();
        any_factor = __syncthreads_or(tid < kPackCtas && *(volatile const int *)(g.odd + tid) != 0);
    } else {
        __syncthreads();
    }
    tc::fence_after();

    // A wait whose answer is the same for all lanes: whether each has found the phase, so that what it waited for may be used.
    auto found = [&](bool mine) -> bool { return __all_sync(0xffffffffu, mine); };
    auto gave_up = [&]() -> bool { return __any_sync(0xffffffffu, *abort_flag != 0); };     // whether a wait of this CTA has
    // A role takes the segments in order from the ring; every warp of it calls this.
    int seg = 0;
    auto take_segment = [&](Segment &sg, int i) -> bool {
        sg = seg_s[i];
        __syncwarp();
        if (lane == 0) tc::arrive(DS4B200_BAR(seg_free, i));
        return sg.t1 >= 0;
    };
    auto next_segment = [&](Segment &sg) -> bool {
        const int i = seg & (kSegRing - 1);
        const bool on = found(tc::wait(DS4B200_BAR(seg_full, i), (uint32_t)((seg / kSegRing) & 1), abort_flag, status));
        ++seg;
        return on && take_segment(sg, i);
    };
    // The same for the warps of a role that meet at named barriers, which have no limit: the first warp waits and says for all whether they go
    // on, so that none stays behind at a barrier.  Two places in turn: a warp writes the next answer only when all have read the last but one.
    auto next_segment_together = [&](Segment &sg, int role, bool first, auto &&sync) -> bool {
        const int i = seg & (kSegRing - 1);
        int *go = &go_s[role][seg & 1];
        if (first) {
            const bool on = found(tc::wait(DS4B200_BAR(seg_full, i), (uint32_t)((seg / kSegRing) & 1), abort_flag, status));
            if (lane == 0) *go = on;
        }
        sync();
        ++seg;
        return *(volatile int *)go != 0 && take_segment(sg, i);
    };

    if (warp >= kLoadWarp0 && warp < kLoadWarp0 + kLoadWarps) {
        // ------------------------------------------------------------------------------ loaders
        // A warp has eight rows of the tile.  Its loads cover two rows at a time, 256 contiguous bytes of each (16 lanes): whole lines,
        // and stores of rows r and r + 1 with their 16-byte units XORed by the row fall on all banks.  Tails go by
        // four lanes per row.  A register is loaded again, with the next unit's bytes, as soon as
        // its value is converted, so loads run a tile ahead of the stores.  A unit is a tile, or 128 or 256 dims of one in f32.
        tc::set_max_registers_up<kLoadRegs>();
        constexpr bool kF32 = FMT == DS4B200_KV_F32, kBlock = FMT == DS4B200_KV_FP8_BLOCK64;
        constexpr int kUnitChunks = !kF32 ? kChunks : (NB % 2 ? 2 : 4), kUnits = kChunks / kUnitChunks;
        constexpr int kSpan = kF32 ? 1 : 4;              // chunks a load of two rows covers (fewer with fewer dims)
        constexpr int kSteps = (kUnitChunks + kSpan - 1) / kSpan, kRegs = kSteps * 4;
        const int lw = warp - kLoadWarp0, r = lw * 8 + (lane >> 2), part = lane & 3;
        const uint32_t row_off = (uint32_t)(r * 128), sw = (uint32_t)(r & 7);
        // of a load of two rows: which one, and the lane's 16 bytes of its 256; eight consecutive lanes (16 with the 8-byte stores
        // of f32 rows) have to fall on all banks
        const int half = kF32 ? lane >> 4 : (lane >> 2) & 1, l16 = kF32 ? lane & 15 : (lane & 3) | ((lane >> 3) << 2);
        const bool tail = kBlock && a.kv.n_rot != 0;
        const int n_scales = kBlock ? (D - a.kv.n_rot) / 64 : 1;
        const int q_row = lw * 8 + ((lane >> 3) & 1), q_lane = (lane & 7) | ((lane >> 4) << 3);     // rows q_row + 2 j, 16 of their bytes
        // The query rows: two at a time, 256 contiguous bytes of each, eight lanes of a row making a 128-byte row of the operand.
        auto query_16 = [&](int64_t row0, int rows, int j, int b) {
            return q_row + 2 * j < rows ? ld_row16(a.q + (row0 + q_row + 2 * j) * D + b * 128 + q_lane * 8) : make_uint4(0, 0, 0, 0);
        };
        auto store_query = [&](const uint4 &x, int j, int b) {
            const int rw = q_row + 2 * j;
            *reinterpret_cast<uint4 *>(q_s + (2 * b + (q_lane >> 3)) * 8192 + rw * 128 + (((uint32_t)(q_lane & 7) ^ (uint32_t)(rw & 7)) << 4)) =
                make_uint4(bf16x2_to_f16x2(x.x), bf16x2_to_f16x2(x.y), bf16x2_to_f16x2(x.z), bf16x2_to_f16x2(x.w));
        };
        // Whether a row's largest value (in amax as two halves per lane) is so far from one that it is scaled; then up and down are its scale.
        auto query_scales = [&](uint32_t (&amax)[4], float (&up)[4], float (&down)[4]) -> bool {
            bool far = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                amax[j] = max(amax[j] & 0xffff0000u, amax[j] << 16);
                far = far || amax[j] < 0x3d800000u || amax[j] > 0x47000000u;
            }
            if (!__any_sync(0xffffffffu, far)) return false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int o = 1; o < 32; o <<= 1)
                    if (o != 8) amax[j] = max(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], o));
                if (amax[j] != 0 && (amax[j] < 0x3d800000u || amax[j] > 0x47000000u)) pow2_parts(__uint_as_float(amax[j]), up[j], down[j]);
            }
            return true;
        };
        auto set_query_scales = [&](const float (&up)[4], int nq) {
            if (q_lane == 0)
#pragma unroll
                for (int j = 0; j < 4; ++j) q_mul[nq & (kScaleSets - 1)][q_row + 2 * j] = up[j] * a.scale * kLog2e;
            __syncwarp();
            if (lane == 0) tc::arrive(DS4B200_BAR(q_full, 0));
        };
        auto load_query = [&](int64_t row0, int rows, int nq) {
            // half a row's dims at a time, as they are where its largest value is within [2^-4, 2^15], else scaled by a power of two in a second pass
            float up[4] = {1.0f, 1.0f, 1.0f, 1.0f}, down[4] = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll 1
            for (int pass = 0; pass < 2; ++pass) {
                uint32_t amax[4] = {0, 0, 0, 0};
#pragma unroll 1
                for (int b0 = 0; b0 < NB; b0 += 2) {
                    uint4 x[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < 2; ++b) x[j][b] = b0 + b < NB ? query_16(row0, rows, j, b0 + b) : make_uint4(0, 0, 0, 0);
                    if (pass == 0 && b0 == 0) tc::wait(DS4B200_BAR(q_free, 0), (uint32_t)((nq & 1) ^ 1), abort_flag, status);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            amax[j] = max_bf16x8(x[j][b], amax[j]);
                            scale_bf16x8(x[j][b], down[j]);
                            if (b0 + b < NB) store_query(x[j][b], j, b0 + b);
                        }
                }
                if (pass || !query_scales(amax, up, down)) break;
            }
            set_query_scales(up, nq);
        };
        if (kPre) {
            // With packed rows these warps fetch the query rows and drain the accumulators, one item apart, while the softmax goes on.
            const int quarter = lw & 3, which = lw >> 2;                    // 32 lanes of tensor memory, 16 of them
            const uint32_t lanes = (uint32_t)(quarter * 32 + which * 16) << 16;
            unsigned char *stage = p_s + 2 * 8192;                          // 32 rows of 128 dims
            auto sync_all = [&]() { asm volatile("bar.sync 4, 256;" ::: "memory"); };
            struct Rows { int64_t row0; int rows; };
            auto take = [&](Rows &it) -> bool {
                Segment sg;
                if (!next_segment_together(sg, 1, lw == 0, sync_all)) return false;
                it = Rows{sg.it.row0, sg.it.rows};
                return true;
            };
            Rows cur{0, 0}, next{0, 0};
            int base = 0;
            bool more = take(next);
            for (int k = -1;; ++k) {
                // the query rows of item k + 1, as they are where a lane's largest value is within [2^-4, 2^15], else scaled by a power of two
                if (more) {
                    uint4 x[4][NB];
                    uint32_t amax[4] = {0, 0, 0, 0};
                    float up[4] = {1.0f, 1.0f, 1.0f, 1.0f}, down[4] = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < NB; ++b) x[j][b] = query_16(next.row0, next.rows, j, b);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < NB; ++b) amax[j] = max_bf16x8(x[j][b], amax[j]);
                    if (query_scales(amax, up, down))
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int b = 0; b < NB; ++b) scale_bf16x8(x[j][b], down[j]);
                    tc::wait(DS4B200_BAR(q_free, 0), (uint32_t)(((k + 1) & 1) ^ 1), abort_flag, status);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < NB; ++b) store_query(x[j][b], j, b);
                    set_query_scales(up, k + 1);
                }
                if (k >= 0) {                                               // item k's accumulators
                    tc::wait(DS4B200_BAR(o_ready, k & (kScaleSets - 1)), (uint32_t)((k / kScaleSets) & 1), abort_flag, status);
                    // Not the last tile's pv_done: with up to 384 dims the products of item k + 1 need nothing of this drain, and two tiles
                    // of them would turn that barrier's parity back.  o_done[k & 1] waits for o_free of item k before its next turn.
                    tc::wait(DS4B200_BAR(o_done, k & 1), (uint32_t)((k >> 1) & 1), abort_flag, status);
                    tc::fence_after();
                    // rolled up: with all blocks unrolled this loop alone was 30 KB, and the instruction fetches of all roles stalled for it
#pragma unroll 1
                    for (int b = 0; b < NB; ++b) {
                        uint32_t o[32];
                        tc::ld_16x64(o_block(base, b) + lanes, o);
                        tc::wait_ld();
                        if (b + 1 == NB || b + 1 == NB - kFree) {
                            tc::fence_before();
                            __syncwarp();
                            if (lane == 0) tc::arrive(b + 1 == NB ? DS4B200_BAR(o_free, k & 1) : DS4B200_BAR(o_half, 0));
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {                       // 32 rows
                            if (h * 32 >= cur.rows) continue;
                            sync_all();                                     // the stage is free
#pragma unroll
                            for (int i = 0; i < 4; i += 2) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float2 f = *reinterpret_cast<const float2 *>(&inv_s[k & (kScaleSets - 1)][h * 32 + 8 * (i + e) + 2 * (lane & 3)]);
                                    const uint32_t *y = &o[16 * h + 4 * (i + e)];
                                    const float2 y0 = mul2(make_float2(__uint_as_float(y[0]), __uint_as_float(y[1])), f);
                                    const float2 y1 = mul2(make_float2(__uint_as_float(y[2]), __uint_as_float(y[3])), f);
                                    w[2 * e] = h2b(y0.x, y0.y);
                                    w[2 * e + 1] = h2b(y1.x, y1.y);
                                }
                                const int rw = 8 * (i + (lane >> 4)) + (lane & 7), unit = quarter * 4 + which * 2 + ((lane >> 3) & 1);
                                asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                                             ::"r"(smem_addr(stage) + rw * 256 + ((unit ^ (rw & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                            }
                            sync_all();
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int rw = i * 16 + lw * 2 + (lane >> 4), unit = lane & 15;
                                if (h * 32 + rw < cur.rows)
                                    __stcs(reinterpret_cast<uint4 *>(a.out + (cur.row0 + h * 32 + rw) * D + b * 128 + unit * 8),
                                           *reinterpret_cast<const uint4 *>(stage + rw * 256 + ((unit ^ (rw & 7)) << 4)));
                            }
                        }
                    }
                }
                if (!more) break;
                if (k >= 0) base = next_base(base);
                cur = next;
                more = take(next);
            }
        } else {
        uint4 v[kRegs];                                  // [step][row pair]
        float sc[kF32 ? 1 : kRegs];                      // the scale of each
        float4 tl[kBlock ? 4 : 1];
        struct Slots { int pair[4], own, rows; };        // of rows 2 j + half, and of row r; tile_rows, -1 also where a wait has given up
        auto slots_of = [&](int n) -> Slots {
            const int i = n & (kTileRing - 1);
            if (!found(tc::wait(DS4B200_BAR(tile_full, i), (uint32_t)((n / kTileRing) & 1), abort_flag, status))) return Slots{{-1, -1, -1, -1}, -1, -1};
            const int4 p = *reinterpret_cast<const int4 *>(&slot_s[kPre ? 0 : i][lw * 8 + half * 4]);
            return Slots{{p.x, p.y, p.z, p.w}, kBlock && tail ? slot_s[kPre ? 0 : i][lw * 8 + ((lane >> 2) & 1) * 4 + (lane >> 3)] : 0, tile_rows[i]};
        };
        auto load = [&](int my, bool all, int unit, int step, int j) {      // all: of the warp's rows exist
            const int k = step * 4 + j;
            if (!all) {
                v[k] = make_uint4(0, 0, 0, 0);
                if (!kF32) sc[kF32 ? 0 : k] = 1.0f;
                if (my < 0) return;
            }
            if (kF32) {
                v[k] = ld_row16(a.kv.raw + (int64_t)my * D + (unit * kUnitChunks + step) * 64 + l16 * 4);
            } else {
                const int c = step * 4 + (l16 >> 2);                // chunk of this lane
                // lanes past the codes load the row's first ones, which nobody stores
                const bool in = c < kChunks && !(tail && c == kChunks - 1);
                v[k] = ld_row16(a.kv.codes + (int64_t)my * D + (in ? step * 256 + l16 * 16 : 0));
                sc[kF32 ? 0 : k] = __ldg(a.kv.scales + (kBlock ? (int64_t)my * n_scales + (in ? c : 0) : (int64_t)my));
            }
        };
        auto load_tail = [&](int my) {
            if (kBlock)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 x = my >= 0 && tail ? ld_row16(a.kv.tail + (int64_t)my * 64 + part * 16 + j * 4) : make_uint4(0, 0, 0, 0);
                    tl[kBlock ? j : 0] = make_float4(__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
                }
        };
        Slots here = slots_of(0);
        if (here.rows >= 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int step = 0; step < kSteps; ++step) load(here.pair[j], false, 0, step, j);
            load_tail(here.own);
        }
        for (int n = 0, nq = 0; here.rows >= 0; ++n) {
            const int buf = n & 1, ring = n & (kTileRing - 1);
            const uint32_t use = (uint32_t)(((n >> 1) & 1) ^ 1);
            unsigned char *dst = k_s + buf * kTileBytes;
            if (here.rows) load_query(tile_row0[ring], here.rows, nq++);    // a segment's query rows come ahead of its first tile
            const Slots next = slots_of(n + 1);          // the tile behind this one
            const bool all_here = kUnits > 1 && __all_sync(0xffffffffu, (here.pair[0] | here.pair[1] | here.pair[2] | here.pair[3]) >= 0);
            const bool all_next = __all_sync(0xffffffffu, (next.pair[0] | next.pair[1] | next.pair[2] | next.pair[3]) >= 0);
            // The MMA warp makes the stores visible to the async proxy: a proxy fence here would wait for the loads in flight.
            auto hand_over = [&](int k) {
                __syncwarp();
                if (lane == 0) tc::arrive(DS4B200_BAR(full, (buf) * 2 + (k)));
            };
            // Rows of ordinary size become f16 as they are (E4M3 codes times a power of two stay exact).  Where one of the warp's rows has
            // a scale outside [2^-17, 2^5] or a tail value beyond 2^14, its rows keep a factor, and the tile is marked for the softmax.
            float down = 1.0f;
            bool bad = false;
            if (!kF32) {
#pragma unroll
                for (int k = 0; k < kRegs; ++k) bad = bad || !(sc[kF32 ? 0 : k] >= 0x1p-17f && sc[kF32 ? 0 : k] <= 0x1p5f);
                if (kBlock)
#pragma unroll
                    for (int j = 0; j < 4; ++j) bad = bad || !(amax4(tl[kBlock ? j : 0]) <= 0x1p14f);
            }
            const bool hole = here.pair[0] == kHole || here.pair[1] == kHole || here.pair[2] == kHole || here.pair[3] == kHole;
            const bool odd = __any_sync(0xffffffffu, bad || hole);
            if (odd) {
                tc::wait(DS4B200_BAR(pv_done, (buf) * 2 + (0)), use, abort_flag, status);       // the softmax has done with this buffer's factors
                if (lane == 0) odd_s[buf] = odd_w[buf][lw] = n + 1;
                float mine = 1.0f;                       // the factor of row r
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float mul = 1.0f;
                    if (!kF32) {
                        float top = sc[kF32 ? 0 : j];
                        if (kSteps > 1) top = fmaxf(top, sc[kF32 || kSteps < 2 ? 0 : 4 + j]);
                        if (kBlock) {                    // over the row's lanes (which differ in bits 0, 1, 3, 4), and its tail
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1)
                                if (o != 4) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            float t4 = 0.0f;
#pragma unroll
                            for (int i = 0; i < 4; ++i) t4 = fmaxf(t4, amax4(tl[kBlock ? i : 0]));
                            t4 = fmaxf(t4, __shfl_xor_sync(0xffffffffu, t4, 1));
                            t4 = fmaxf(t4, __shfl_xor_sync(0xffffffffu, t4, 2));
                            top = fmaxf(top, __shfl_sync(0xffffffffu, t4, (2 * j + half) * 4) * (1.0f / 256.0f));
                        }
                        // not below kLeast: the weight times the factor would leave f32's range while the weight still counts
                        mul = top < kLeast ? kLeast : top;
                        float inv = 1.0f / mul;
                        if (kBlock) pow2_parts(top == 0.0f ? top : mul, mul, inv);
#pragma unroll
                        for (int st = 0; st < kSteps; ++st) sc[kF32 ? 0 : st * 4 + j] = kBlock || top < kLeast ? sc[kF32 ? 0 : st * 4 + j] * inv : 1.0f;
                    }
                    const float got = __shfl_sync(0xffffffffu, mul, kF32 ? (lane & 4) << 2 : lane & 4);   // of a lane whose half is row r's parity
                    if ((lane >> 3) == j) mine = got;
                    if (l16 == 0) {
                        const int rw = lw * 8 + 2 * j + half;
                        row_fma[buf][2 * (rw & ~1) + (rw & 1)] = mul;
                        row_fma[buf][2 * (rw & ~1) + 2 + (rw & 1)] = here.pair[j] >= 0 ? __log2f(mul) : -INFINITY;
                        row_div[buf][rw] = mul == mul ? 1.0f / mul : 1.0f;
                    }
                }
                if (kBlock) down = 1.0f / mine;
            }
            // A scale of a whole row is any number, and below 2^-14 f16 would keep too few of its bits (2^-8 of it at 2^-17): such a row's codes take
            // 2^8 times it, and 2^-8 behind that, which costs at most half of f16's smallest step.
            bool fine = false;
            if (FMT == DS4B200_KV_FP8_ROW) {
#pragma unroll
                for (int j = 0; j < 4; ++j) fine = fine || sc[kF32 ? 0 : j] < 0x1p-14f;
                fine = __any_sync(0xffffffffu, fine) && !odd;
            }
            uint32_t spoilt = 0;                         // bit j: row 2 j + half has a value that is not finite
            const int rw = lw * 8 + half;
#pragma unroll
            for (int unit = 0; unit < kUnits; ++unit)
#pragma unroll
                for (int step = 0; step < kSteps; ++step) {
                    const int c0 = unit * kUnitChunks + step * kSpan;       // first chunk of the step
                    if (c0 == 0) tc::wait(DS4B200_BAR(pv_done, (buf) * 2 + (0)), use, abort_flag, status);
                    if (kParts > 1 && c0 == 2 * kPart0) {
                        hand_over(0);
                        tc::wait(DS4B200_BAR(pv_done, (buf) * 2 + (kParts - 1)), use, abort_flag, status);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 x = v[step * 4 + j];
                        const uint32_t r7 = (uint32_t)(2 * j + half);
                        if (kF32) {
                            uint32_t o[2] = {sat_h2(__uint_as_float(x.x), __uint_as_float(x.y)), sat_h2(__uint_as_float(x.z), __uint_as_float(x.w))};
                            if (SHARED && several) spoilt |= (uint32_t)drop_nonfinite(o) << j;
                            *reinterpret_cast<uint2 *>(dst + c0 * 8192 + (rw + 2 * j) * 128 + ((((uint32_t)l16 >> 1) ^ r7) << 4) + (l16 & 1) * 8) =
                                make_uint2(o[0], o[1]);
                        } else {
                            const int c = c0 + (l16 >> 2);
                            const float scale = sc[kF32 ? 0 : step * 4 + j];
                            const bool up = fine && scale < 0x1p-14f;
                            const __half2 f = __float2half2_rn(up ? scale * 0x1p8f : scale);
                            uint32_t o[8];
                            const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) e4m3x4(y[k], o[2 * k], o[2 * k + 1]);
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = h2_bits(__hmul2(*reinterpret_cast<__half2 *>(&o[k]), f));
                            if (FMT == DS4B200_KV_FP8_ROW && fine) {
                                const __half2 back = __float2half2_rn(up ? 0x1p-8f : 1.0f);
#pragma unroll
                                for (int k = 0; k < 8; ++k) o[k] = h2_bits(__hmul2(*reinterpret_cast<__half2 *>(&o[k]), back));
                            }
                            if (c < kChunks && !(tail && c == kChunks - 1)) {
                                if (SHARED && several) spoilt |= (uint32_t)drop_nonfinite(o) << j;
                                unsigned char *to = dst + c * 8192 + (rw + 2 * j) * 128;
                                const uint32_t u = (uint32_t)(l16 & 3) * 2;
                                *reinterpret_cast<uint4 *>(to + ((u ^ r7) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                                *reinterpret_cast<uint4 *>(to + (((u + 1) ^ r7) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                            }
                        }
                        if (unit + 1 < kUnits) load(here.pair[j], all_here, unit + 1, step, j);
                        else if (next.rows >= 0) load(next.pair[j], all_next, 0, step, j);
                    }
                }
            if (kBlock && tail) {
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 y = tl[kBlock ? j : 0];
                    o[2 * j] = h2_bits(__floats2half2_rn(y.x * down, y.y * down));
                    o[2 * j + 1] = h2_bits(__floats2half2_rn(y.z * down, y.w * down));
                }
                if (SHARED && several) {                 // row r's flag goes to the lanes that have it as 2 j + half
                    const uint32_t rows_bad = __ballot_sync(0xffffffffu, drop_nonfinite(o));
#pragma unroll
                    for (int j = 0; j < 4; ++j) spoilt |= (rows_bad >> (4 * (2 * j + half)) & 15u ? 1u : 0u) << j;
                }
                unsigned char *to = dst + (kChunks - 1) * 8192 + row_off;
                *reinterpret_cast<uint4 *>(to + (((uint32_t)(part * 2) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4 *>(to + (((uint32_t)(part * 2 + 1) ^ sw) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                if (next.rows >= 0) load_tail(next.own);
            }
            // Several tokens share the tile, and 0 * NaN would reach the ones that do not see the row: it has zeros where it is not finite, and
            // the factor NaN for those that see it.
            if (SHARED && several && __any_sync(0xffffffffu, spoilt != 0)) {
                if (lane == 0) odd_s[buf] = odd_w[buf][lw] = n + 1;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t who = __ballot_sync(0xffffffffu, spoilt >> j & 1);
                    const bool is = (who & (kF32 ? 0xffffu << (16 * half) : 0x0f0f0f0fu << (4 * half))) != 0;     // any lane of the row
                    if (l16 == 0 && (is || !odd)) {
                        const int k = rw + 2 * j;
                        row_fma[buf][2 * (k & ~1) + (k & 1)] = is ? __uint_as_float(0x7fffffffu) : 1.0f;
                        if (!odd) row_fma[buf][2 * (k & ~1) + 2 + (k & 1)] = 0.0f;
                        if (!odd) row_div[buf][k] = 1.0f;
                    }
                }
            }
            hand_over(kParts - 1);
            if (lane == 0) tc::arrive(DS4B200_BAR(tile_free, ring));
            here = next;
        }
        }
    } else if (warp >= kMmaWarp) {
        tc::set_max_registers_down<kOtherRegs>();
        const uint32_t one = tc::elect();
        const uint32_t k_desc = tc::desc_lo(smem_addr(k_s), 0);
        if (warp == kMmaWarp) {
            // -------------------------------------------------------------------------- S = Q K^T
            const uint32_t q_desc = tc::desc_lo(smem_addr(q_s), 0);
            Segment sg;
            int n = 0;
            for (int nq = 0; next_segment(sg); ++nq) {
                const int t0 = __shfl_sync(0xffffffffu, sg.t0, 0), t1 = __shfl_sync(0xffffffffu, sg.t1, 0);
                const int n_rows = __shfl_sync(0xffffffffu, sg.it.n, 0), na = __shfl_sync(0xffffffffu, sg.it.na, 0), ta = (na + 63) >> 6;
                tc::wait<20>(DS4B200_BAR(q_full, 0), (uint32_t)(nq & 1), abort_flag, status);
                for (int t = t0; t < t1; ++t, ++n) {
                    const int buf = n & 1;
                    const uint32_t phase = (uint32_t)((n >> 1) & 1), k0 = k_desc + (uint32_t)(buf * (kTileBytes >> 4));
                    const int groups = min(max(((t < ta ? na - 64 * t : n_rows - na - 64 * (t - ta)) + 15) >> 4, 1), 4);      // of 16 cache rows
                    const uint32_t idesc = tc::idesc_f16(64, 0, false) | (uint32_t)groups << 18;
                    tc::wait<20>(DS4B200_BAR(s_free, buf), phase ^ 1, abort_flag, status);
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        tc::wait<20>(DS4B200_BAR(full, (buf) * 2 + (part)), phase, abort_flag, status);
                        tc::fence_async();               // for the loaders' stores, of the query rows too
                        tc::fence_after();
#pragma unroll 1
                        for (int c = part * 2 * kPart0; c < (part + 1 == kParts ? kChunks : 2 * kPart0); ++c)
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)
                                tc::mma_f16(one, s_tmem + buf * 64, q_desc + (uint32_t)(c * 512 + ks * 2), k0 + (uint32_t)(c * 512 + ks * 2), idesc,
                                            c > 0 || ks > 0);
                    }
                    tc::commit(one, DS4B200_BAR(s_full, buf));
                }
                tc::commit(one, DS4B200_BAR(q_free, 0));
            }
            if (gave_up()) { tc::commit(one, DS4B200_BAR(quiet, 0)); tc::settle(DS4B200_BAR(quiet, 0), 0); }
        } else if (warp == kMmaWarp + 1) {
            // -------------------------------------------------------------------------- O^T += V^T P^T
            const uint32_t v_desc = tc::desc_lo(smem_addr(k_s), 8192), p_desc = tc::desc_lo(smem_addr(p_s), 0);
            constexpr uint32_t idesc = tc::idesc_f16(128, 64, true);
            uint32_t scaled_uses[2] = {0, 0};
            auto scaled_phase = [&](int b) { return scaled_uses[b]++ & 1; };
            Segment sg;
            int n = 0;
            int base = 0;
            for (int k = 0; next_segment(sg); ++k, base = next_base(base)) {
                const int t0 = __shfl_sync(0xffffffffu, sg.t0, 0), t1 = __shfl_sync(0xffffffffu, sg.t1, 0);
                if (kPre && k > 1) tc::wait<20>(DS4B200_BAR(o_free, k & 1), (uint32_t)(((k - 2) >> 1) & 1), abort_flag, status);
                const int n_rows = __shfl_sync(0xffffffffu, sg.it.n, 0), na = __shfl_sync(0xffffffffu, sg.it.na, 0), ta = (na + 63) >> 6;
                for (int t = t0; t < t1; ++t, ++n) {
                    const int buf = n & 1;
                    const uint32_t v0 = v_desc + (uint32_t)(buf * (kTileBytes >> 4)), p0 = p_desc + (uint32_t)(buf * 512);
                    const int groups = min(max(((t < ta ? na - 64 * t : n_rows - na - 64 * (t - ta)) + 15) >> 4, 1), 4);
                    tc::wait<20>(DS4B200_BAR(p_full, buf), (uint32_t)((n >> 1) & 1), abort_flag, status);
                    if (*(volatile int *)&grown_s[buf] == n + 1) tc::wait<20>(DS4B200_BAR(scaled, buf), scaled_phase(buf), abort_flag, status);
                    tc::fence_async();
                    tc::fence_after();
#pragma unroll 1
                    for (int m = 0; m < NB; ++m) {
                        if (kPre && kFree < NB && m == kFree && t == t0 && k > 0) {
                            tc::wait<20>(DS4B200_BAR(o_half, 0), (uint32_t)((k - 1) & 1), abort_flag, status);
                            tc::fence_after();
                        }
                        const uint32_t o_m = __shfl_sync(0xffffffffu, o_block(base, m), 0);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            if (ks < groups)
                                tc::mma_f16(one, o_m, v0 + (uint32_t)(m * 1024 + ks * 128), p0 + (uint32_t)(ks * 2), idesc, t > t0 || ks > 0);
                        if (kParts > 1 && m == kPart0 - 1) tc::commit(one, DS4B200_BAR(pv_done, (buf) * 2 + (0)));
                    }
                    tc::commit(one, DS4B200_BAR(pv_done, (buf) * 2 + (kParts - 1)));
                }
                if (kPre) tc::commit(one, DS4B200_BAR(o_done, k & 1));
            }
            if (gave_up()) { tc::commit(one, DS4B200_BAR(quiet, 1)); tc::settle(DS4B200_BAR(quiet, 1), 0); }
        } else if (warp == kMmaWarp + 2) {
            // -------------------------------------------------------------------------- schedule
            int slot = g.split ? start_slot : (int)blockIdx.x, tile = g.split ? start_tile : 0;
            const int step = g.split ? 1 : (int)gridDim.x;
            int longest = 0;                             // it waits for whole items, 16 polls of 0.3 us a tile at most
            for (bool end = false; !end; ++seg) {
                Segment sg;
                sg.t0 = 0;
                sg.t1 = -1;
                end = true;
                while (left > 0 && slot < g.n_slots) {
                    sg.it = get_item<kPre>(a, g.group, g.head_groups, slot);
                    slot += step;
                    if (sg.it.tiles == 0) continue;
                    longest = max(longest, sg.it.tiles);
                    sg.t0 = tile;
                    sg.t1 = (int)min((long long)sg.it.tiles, tile + left);
                    tile = 0;
                    if (g.split) left -= sg.t1 - sg.t0;
                    end = false;
                    break;
                }
                const int i = seg & (kSegRing - 1);
                // (without the phase the place may still be read)
                if (!found(tc::wait<300>(DS4B200_BAR(seg_free, i), (uint32_t)(((seg / kSegRing) & 1) ^ 1), abort_flag, status, tc::kWaitPolls + 16 * longest)) ||
                    gave_up()) break;
                if (lane == 0) {
                    if (kPre && !end) prefetch_l2(a.q + sg.it.row0 * D, sg.it.rows * D * 2);     // some items before they are wanted
                    seg_s[i] = sg;
                    tc::arrive(DS4B200_BAR(seg_full, i));
                }
                __syncwarp();
            }
        } else if (kPre) {
            // -------------------------------------------------------------------------- copy packed rows
            Segment sg;
            int n = 0, sent = 0;                         // parts of tiles
            bool stop = false;
            while (!stop && next_segment(sg)) {
                for (int t = sg.t0; t < sg.t1 && !stop; ++t, ++n) {
                    const int buf = n & 1, ta = first_run_tiles(sg.it);
                    const int from = t < ta ? sg.it.at_a + 64 * t : sg.it.at_b + 64 * (t - ta);
                    // up to 16 rows (the MMAs read no more of them either), e.g. the first rows beside a window of 128
                    const bool few = rows_in_tile(sg.it, t) <= 16;
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        stop = !found(tc::wait<20>(DS4B200_BAR(pv_done, buf * 2 + part), (uint32_t)(((n >> 1) & 1) ^ 1), abort_flag, status)) || stop;
                        if (stop) continue;              // the last copy to this place may be in flight
                        ++sent;
                        if (lane == 0) {
                            constexpr int kFirst = kParts > 1 ? 2 * kPart0 : kChunks;
                            const int c0 = part * kFirst, c1 = part ? kChunks : kFirst;
                            tc::expect(DS4B200_BAR(full, buf * 2 + part), (uint32_t)(c1 - c0) * (few ? 2048u : 8192u));
                            for (int c = c0; c < c1; ++c)
                                tc::load_box(smem_addr(k_s) + buf * kTileBytes + c * 8192, few ? &g.few : &g.rows, c * 64, from, DS4B200_BAR(full, buf * 2 + part));
                        }
                        __syncwarp();
                    }
                }
            }
            if (gave_up())                               // no copy is in flight when the kernel ends
                for (int q = max(sent - 2 * kParts, 0); q < sent; ++q) {
                    const int k = q / kParts;
                    tc::settle(DS4B200_BAR(full, (k & 1) * 2 + q % kParts), (uint32_t)((k >> 1) & 1));
                }
        } else {
            // -------------------------------------------------------------------------- find
            // The pool rows of the tiles to come, two per lane, up to kTileRing tiles ahead of the loaders: a page-table entry, and the first
            // touch of a page, take a few thousand cycles, so the rows' lines are fetched into L2 ahead of the loads.
            constexpr bool kF32 = FMT == DS4B200_KV_F32, kBlock = FMT == DS4B200_KV_FP8_BLOCK64;
            const bool tail = kBlock && a.kv.n_rot != 0;
            Segment sg;
            int n = 0;
            for (bool more = true; more;) {
                sg.t0 = 0;
                more = next_segment(sg);
                const int t1 = more ? sg.t1 : sg.t0 + 1;                    // one more entry says that it ends
                for (int t = sg.t0; t < t1; ++t, ++n) {
                    const int i = n & (kTileRing - 1);
                    // without the phase the place may still be read
                    if (!found(tc::wait<300>(DS4B200_BAR(tile_free, i), (uint32_t)(((n / kTileRing) & 1) ^ 1), abort_flag, status))) { more = false; break; }
                    if (lane == 0) {
                        tile_rows[i] = !more ? -1 : t == sg.t0 ? sg.it.rows : 0;
                        tile_row0[i] = sg.it.row0;
                    }
                    int slot[2] = {-1, -1};
                    if (more) {
                        int page[2], in[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int k = t * kRows + lane + 32 * h, at = k < sg.it.first ? k : sg.it.lo + (k - sg.it.first);
                            const int pg = g.page_shift >= 0 ? at >> g.page_shift : at / a.kv.page_rows;
                            in[h] = at - pg * a.kv.page_rows;
                            page[h] = k < sg.it.n ? max(__ldg(a.page_table + sg.it.b * a.table_width + pg), -1) : -2;
                            if (SHARED) row_at[kPre || !SHARED ? 0 : n & (2 * kTileRing - 1)][lane + 32 * h] = at;
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            slot[h] = page[h] == -2 ? -1 : page[h] >= 0 && page[h] < a.kv.n_pages ? page[h] * a.kv.page_rows + in[h] : kHole;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = lane + 32 * h;                        // loaders read the even or the odd rows of eight
                        slot_s[kPre ? 0 : i][(r & ~7) + (r & 1) * 4 + ((r & 7) >> 1)] = slot[h];
                        // one prefetch per run of neighbours in the pool: 64 of them a tile kept the copy engine busier than the loaders
                        const int before = __shfl_up_sync(0xffffffffu, slot[h], 1);
                        const uint32_t heads = __ballot_sync(0xffffffffu, lane == 0 || slot[h] < 0 || slot[h] != before + 1);
                        if (!kF32 && (heads >> lane & 1) && slot[h] >= 0) {     // f32 rows: 2 KiB of loads in flight a row do better alone (96 sequences 82 us, 68)
                            const uint32_t behind = lane == 31 ? 0 : heads >> (lane + 1);
                            const int run = behind ? __ffs(behind) : 32 - lane;
                            const int64_t sl = slot[h];
                            prefetch_l2(a.kv.codes + sl * D, run * D);
                            if (tail) prefetch_l2(a.kv.tail + sl * 64, run * 256);
                        }
                    }
                    if (more && t == sg.t0 && lane == 0) prefetch_l2(a.q + sg.it.row0 * D, sg.it.rows * D * 2);    // the segment's query rows
                    __syncwarp();
                    if (lane == 0) tc::arrive(DS4B200_BAR(tile_full, i));
                }
            }
        }
    } else {
        // ------------------------------------------------------------------------------ softmax and output
        // Eight warps, two per quarter of tensor memory's lanes: a quarter holds 16 rows of S (lanes 0-15), of which each warp takes
        // eight, four lanes and 16 columns each.
        tc::set_max_registers_down<kSoftRegs>();
        const int quarter = warp & 3, group = warp >> 2;
        const int row = quarter * 16 + group * 8 + (lane >> 2);
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        unsigned char *stage = p_s + group * 8192;      // of this group's output, where its weights' buffers are free
        // One warp polls the barriers of the MMAs, the others wait for it here: the hardware's barrier costs them no issue slots.
        auto sync_all = [&]() { asm volatile("bar.sync 3, 256;" ::: "memory"); };
        auto sync_group = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
        Meta last{0, 0, 0, 0, 0};
        Segment sg;
        int n = 0;
        long long done = 0;
        int base = 0;
        for (int nq = 0; next_segment_together(sg, 0, warp == 0, sync_all); ++nq, base = next_base(base)) {
            const Item &it = sg.it;
            float qk = 0.0f, m = -INFINITY;
            float2 l = make_float2(0.0f, 0.0f);
            const int p = it.p0 + (several ? row / a.n_heads : 0);
            const int from = a.window > 0 ? p - a.window : -1;              // cache rows above it are in the window
            // Scales the accumulators ahead of tile k's product where a row of that tile asked for it; behind a sync_all().
            auto follow = [&](int k) {
                const int buf = k & 1;
                if (*(volatile int *)&grown_s[buf] != k + 1) return;
                tc::wait(DS4B200_BAR(pv_done, (buf ^ 1) * 2 + (kParts - 1)), (uint32_t)(((k - 1) >> 1) & 1), abort_flag, status);
                tc::fence_after();
#pragma unroll 1
                for (int u = group; u < NB * 4; u += 2) {
                    uint32_t o[16];
                    const uint32_t at = o_block(base, u >> 2) + (u & 3) * 16 + lane_base;
                    tc::ld16(at, o);
                    tc::wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fac_s[buf][(u & 3) * 16 + i]);
                    tc::st16(at, o);
                }
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive(DS4B200_BAR(scaled, buf));
            };
            for (int t = sg.t0; t < sg.t1; ++t, ++n) {
                const int buf = n & 1;
                const uint32_t phase = (uint32_t)((n >> 1) & 1);
                if (warp == 0) {
                    tc::wait<20>(DS4B200_BAR(full, (buf) * 2 + (kParts - 1)), phase, abort_flag, status);
                    tc::wait<20>(DS4B200_BAR(s_full, buf), phase, abort_flag, status);
                }
                sync_all();
                if (t > sg.t0) follow(n - 1);
                tc::fence_after();
                uint32_t x[32];
                tc::ld_16x64(s_tmem + buf * 64 + lane_base, x);
                // written ahead of the segment's first tile by the same warps; q_full itself may be phases ahead of this warp
                if (t == sg.t0) qk = q_mul[nq & (kScaleSets - 1)][row];
                tc::wait_ld();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive(DS4B200_BAR(s_free, buf));
                float2 v[8];
                const float2 k2 = make_float2(qk, qk);
                const bool odd = kPre ? any_factor : *(volatile int *)&odd_s[buf] == n + 1;
                const float *fac = nullptr;              // of the tile's packed rows
                if (kPre) fac = g.fac + (t < first_run_tiles(it) ? it.at_a + 64 * t : it.at_b + 64 * (t - first_run_tiles(it)));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (group) v[i] = mul2(make_float2(__uint_as_float(x[4 * i + 2]), __uint_as_float(x[4 * i + 3])), k2);
                    else v[i] = mul2(make_float2(__uint_as_float(x[4 * i]), __uint_as_float(x[4 * i + 1])), k2);
                }
                if (odd) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {                          // column block i is loader i's
                        if (kPre) {
                            const float f0 = fac[8 * i + 2 * (lane & 3)], f1 = fac[8 * i + 2 * (lane & 3) + 1];
                            v[i] = fma2(v[i], make_float2(f0, f1), make_float2(__log2f(f0), __log2f(f1)));
                            continue;
                        }
                        if (odd_w[buf][i] != n + 1) continue;
                        const float4 f = *reinterpret_cast<const float4 *>(&row_fma[buf][2 * (8 * i + 2 * (lane & 3))]);
                        v[i] = fma2(v[i], make_float2(f.x, f.y), make_float2(f.z, f.w));
                    }
                }
                if (rows_in_tile(it, t) < kRows) {       // columns past the rows: S was not computed there
                    const int end = rows_in_tile(it, t) - 2 * (lane & 3);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (8 * i >= end) v[i].x = -INFINITY;
                        if (8 * i + 1 >= end) v[i].y = -INFINITY;
                    }
                }
                if (several) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        int2 at;
                        if (kPre) {
                            at.x = (t < first_run_tiles(it) ? it.lo + 64 * t : 64 * (t - first_run_tiles(it))) + 8 * i + 2 * (lane & 3);
                            at.y = at.x + 1;
                        } else {
                            at = *reinterpret_cast<const int2 *>(&row_at[kPre || !SHARED ? 0 : n & (2 * kTileRing - 1)][8 * i + 2 * (lane & 3)]);
                        }
                        if (at.x > p || (at.x <= from && at.x >= a.n_first)) v[i].x = -INFINITY;
                        if (at.y > p || (at.y <= from && at.y >= a.n_first)) v[i].y = -INFINITY;
                    }
                }
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i + 4].x, v[i + 4].y));
                float top = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])), f = 1.0f;
                // A row keeps the reference its maximum had until one of its values lies kRescale above it.  Then it takes a
                // new one, and every row's factor for the accumulators (a column of O^T) is left for follow(), which the
                // warps run together, at the next tile.
                if (__any_sync(0xffffffffu, !(top <= m + kRescale))) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (m > -INFINITY && top > m + kRescale) {
                        f = tc::exp2_approx(m - top);
                        m = top;
                        l = mul2(l, make_float2(f, f));
                        grown_s[buf] = n + 1;
                    }
                    if (m == -INFINITY) m = top;
                }
                if ((lane & 3) == 0) fac_s[buf][row] = f;
                const float ref = m == -INFINITY ? 0.0f : -m;
                const float2 ref2 = make_float2(ref, ref), lift2 = make_float2(kLift, kLift);
                // Weights are stored as kLift times what they are relative to the reference: down to 2^-21 of it they are normal f16 numbers, smaller
                // ones are off by 2^-32 of it (without the lift 2^-25, which 131072 rows can add up to 2^-8).
                unsigned char *dst = p_s + buf * 8192 + row * 128 + (lane & 3) * 4;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = add2(v[i], ref2);
                    v[i].x = tc::exp2_approx(v[i].x);
                    v[i].y = tc::exp2_approx(v[i].y);
                    const float2 y = mul2(v[i], lift2);
                    *reinterpret_cast<uint32_t *>(dst + (((uint32_t)i ^ (uint32_t)(row & 7)) << 4)) = h2_bits(__floats2half2_rn(y.x, y.y));
                }
                if (odd) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (kPre) {
                            const float f0 = fac[8 * i + 2 * (lane & 3)], f1 = fac[8 * i + 2 * (lane & 3) + 1];
                            // A column past the rows has the weight 0 and whatever its factor's place holds: only a factor that the
                            // packing can have left (0, NaN, kLeast and above) has a reciprocal whose product with 0 is 0.
                            v[i] = mul2(v[i], make_float2(f0 >= kLeast ? __fdividef(1.0f, f0) : 0.0f, f1 >= kLeast ? __fdividef(1.0f, f1) : 0.0f));
                        } else if (odd_w[buf][i] == n + 1) v[i] = mul2(v[i], *reinterpret_cast<const float2 *>(&row_div[buf][8 * i + 2 * (lane & 3)]));
                }
                l = add2(l, add2(add2(add2(v[0], v[1]), add2(v[2], v[3])), add2(add2(v[4], v[5]), add2(v[6], v[7]))));
                tc::fence_async();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive(DS4B200_BAR(p_full, buf));
            }
            sync_all();
            follow(n - 1);
            float sum = l.x + l.y;
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const bool whole = sg.t0 == 0 && sg.t1 == it.tiles;
            const int part = 2 * (int)blockIdx.x + (sg.t0 == 0 ? 1 : 0);
            float inv = 1.0f, lse = 0.0f;
            if (whole) {
                float lse2 = sum > 0.0f ? m + __log2f(sum) : (sum == sum ? -INFINITY : sum);
                lse = lse2 * (1.0f / kLog2e);
                if (a.sink && row < it.rows) {
                    const float own = lse2, sink = __ldg(a.sink + it.h0 + (several ? row % a.n_heads : row)), s2 = sink_log2(sink);
                    const bool heavy = s2 >= own;        // then the sum is the sink and a little
                    const float hi = heavy ? s2 : own, more = __log2f(1.0f + tc::exp2_approx((heavy ? own : s2) - hi));
                    lse2 = hi + more;
                    lse = heavy ? sink + more * (1.0f / kLog2e) : lse2 * (1.0f / kLog2e);
                }
                inv = m == -INFINITY ? 0.0f : tc::exp2_approx(m - lse2) * (1.0f / kLift);
            }
            if (kPre) {                                  // the loaders drain the accumulators
                if ((lane & 3) == 0) {
                    if (a.lse && row < it.rows) a.lse[it.row0 + row] = lse;
                    inv_s[nq & (kScaleSets - 1)][row] = inv;
                }
                __syncwarp();
                if (lane == 0) tc::arrive(DS4B200_BAR(o_ready, nq & (kScaleSets - 1)));
                continue;
            }
            // the segment's accumulators
            if (warp == 0) tc::wait<20>(DS4B200_BAR(pv_done, ((n - 1) & 1) * 2 + (kParts - 1)), (uint32_t)(((n - 1) >> 1) & 1), abort_flag, status);
            tc::fence_after();
            if ((lane & 3) == 0) {
                if (!whole) g.part_ml[part * kRows + row] = make_float2(m, sum);
                else if (a.lse && row < it.rows) a.lse[it.row0 + row] = lse;
                inv_s[0][row] = inv;
            }
            sync_all();
            tc::fence_after();
            // In tensor memory a lane is a dim and a column a query row.
            if (whole) {
                // 128 dims of 32 rows at a time through the weights' buffers, which are free here: stmatrix turns 8 x 8 blocks around, rows
                // of 256 bytes with their 16-byte units XORed by the row, and every lane stores 16 bytes of a row
#pragma unroll 1
                for (int u = group; u < NB * 2; u += 2) {
                    const int b = u >> 1, r0 = (u & 1) * 32;
                    if (r0 >= it.rows) continue;
                    uint32_t o[2][16];
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)                          // 16 of the warp's 32 dims
                        tc::ld_16x32(o_tmem + b * 64 + r0 + lane_base + ((uint32_t)(hh * 16) << 16), o[hh]);
                    tc::wait_ld();
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const float2 f0 = *reinterpret_cast<const float2 *>(&inv_s[0][r0 + 8 * i + 2 * (lane & 3)]);
                        const float2 f1 = *reinterpret_cast<const float2 *>(&inv_s[0][r0 + 8 * i + 8 + 2 * (lane & 3)]);
                        const int rw = 8 * (i + (lane >> 4)) + (lane & 7);
#pragma unroll
                        for (int hh = 0; hh < 2; ++hh) {
                            const uint32_t *y = &o[hh][4 * i];
                            uint32_t w[4];
                            w[0] = h2b(__uint_as_float(y[0]) * f0.x, __uint_as_float(y[1]) * f0.y);
                            w[1] = h2b(__uint_as_float(y[2]) * f0.x, __uint_as_float(y[3]) * f0.y);
                            w[2] = h2b(__uint_as_float(y[4]) * f1.x, __uint_as_float(y[5]) * f1.y);
                            w[3] = h2b(__uint_as_float(y[6]) * f1.x, __uint_as_float(y[7]) * f1.y);
                            const int unit = quarter * 4 + hh * 2 + ((lane >> 3) & 1);
                            asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                                         ::"r"(smem_addr(stage) + rw * 256 + ((unit ^ (rw & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        }
                    }
                    sync_group();
                    const int t128 = tid & 127, unit = t128 & 15;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rw = i * 8 + (t128 >> 4);
                        if (r0 + rw < it.rows)
                            __stcs(reinterpret_cast<uint4 *>(a.out + (it.row0 + r0 + rw) * D + b * 128 + unit * 8),
                                   *reinterpret_cast<const uint4 *>(stage + rw * 256 + ((unit ^ (rw & 7)) << 4)));
                    }
                    sync_group();
                }
                sync_all();                                                 // the next weights go where either group's rows were
            } else {
#pragma unroll 1
                for (int u = group; u < NB * 4; u += 2) {
                    const int b = u >> 2, col = (u & 3) * 16;
                    if (col >= it.rows) continue;
                    uint32_t o[16];
                    tc::ld16(o_tmem + b * 64 + col + lane_base, o);
                    tc::wait_ld();
                    float *to = g.part_o + ((int64_t)part * kRows + col) * D + b * 128 + quarter * 32 + lane;
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (col + k < it.rows) to[k * D] = __uint_as_float(o[k]);
                }
            }
            tc::fence_before();
            if (sg.t0 == 0 && sg.t1 < it.tiles)
                last = Meta{it.row0, it.rows, it.h0, (int)((per * (long long)blockIdx.x + done + it.tiles - 1) / per) - (int)blockIdx.x + 1, 0};
            done += sg.t1 - sg.t0;
        }
        if (g.split && tid == 0) g.meta[blockIdx.x] = last;
    }
    tc::fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_s));
}

// Joins the parts of the items that a CTA began and did not finish, in order: with M the largest of the parts' maxima and the sink,
// out = sum_k 2^(m_k - M) O_k / (sum_k 2^(m_k - M) l_k + 2^(sink - M)).  What a unit costs is the latency of its loads, so a unit
// issues its first parts' sums ahead of the statistics that weigh them, and the items' descriptions are in shared memory.
// Few parts: a warp per query row, two parts at a time.  Many (a session of 131072 rows leaves 148 of 128 KiB): a CTA per row and 128
// dims, or per row where rows are many, whose warps take every eighth part.  Alone: 7.3 us (one session of 131072 rows), 8.4 (7 of up to 9001; 11.3 with slices), 8.0
// (64 of up to 16384), 6.0 (96 of 16 heads); with the statistics ahead of the loads, and 64 registers, 11 to 17.
constexpr int kJoinCtas = 4 * kCtas, kJoinWarps = 8, kJoinFew = 8;
static_assert(kCtas <= kJoinWarps * 32, "a thread per part");

// Four partial sums, read once: no place in L1 (up to 0.7 us of a join), and not through the read-only path, since the kernel that writes them has
// not ended when the join becomes resident.
__device__ __forceinline__ float4 ld_part(const float *p) {
    float4 v;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void add_scaled(float4 &o, float w, const float4 &x) {
    o = make_float4(fmaf(w, x.x, o.x), fmaf(w, x.y, o.y), fmaf(w, x.z, o.z), fmaf(w, x.w, o.w));
}

__global__ void __launch_bounds__(kJoinWarps * 32, 3) attn_join_kernel(const AttnArgs a, const Meta *meta, const float2 *part_ml, const float *part_o) {
    __shared__ Meta items[kCtas];
    __shared__ int begun[2][kCtas], n_begun[2];          // items of few and of many parts
    __shared__ float weight[kCtas], most_s[kJoinWarps], sum_s[kJoinWarps];
    __shared__ float4 sums[4][kJoinWarps][32];
    const int D = a.kv.head_dim, slices = D / 128, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    wait_dependency();
    if (tid < kCtas) items[tid] = meta[tid];
    __syncthreads();
    if (warp < 2) {
        int n = 0;
        for (int base = 0; base < kCtas; base += 32) {
            const int c = base + lane, parts = c < kCtas ? items[c].parts : 0;
            const bool is = parts >= 2 && (parts > kJoinFew) == (warp == 1);
            const uint32_t all = __ballot_sync(0xffffffffu, is);
            if (is) begun[warp][n + __popc(all & ((1u << lane) - 1))] = c;
            n += __popc(all);
        }
        if (lane == 0) n_begun[warp] = n;
    }
    __syncthreads();
    auto part_of = [](int c, int k) { return k == 0 ? 2 * c + 1 : 2 * (c + k); };
    auto sink_of = [&](const Meta &it, int row) { return a.sink ? __ldg(a.sink + it.h0 + row % a.n_heads) : -INFINITY; };
    // of a sum l relative to 2^top
    auto lse_of = [](float l, float top, float sink, float sink2) {
        return l == 0.0f ? -INFINITY : sink2 == top ? sink + __log2f(l) * (1.0f / kLog2e) : (top + __log2f(l)) * (1.0f / kLog2e);
    };

    for (int u = blockIdx.x * kJoinWarps + warp; u < n_begun[0] * kRows; u += gridDim.x * kJoinWarps) {
        const int c = begun[0][u / kRows], row = u % kRows;
        const Meta it = items[c];
        if (row >= it.rows) continue;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < it.parts) ml = part_ml[part_of(c, lane) * kRows + row];
        const float sink = sink_of(it, row), sink2 = a.sink ? sink_log2(sink) : -INFINITY;
        float4 x[2][4], o[4];
        auto load = [&](int k) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    x[j][s] = k + j < it.parts && s < slices
                                  ? ld_part(part_o + ((int64_t)part_of(c, k + j) * kRows + row) * D + s * 128 + lane * 4)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        load(0);
#pragma unroll
        for (int s = 0; s < 4; ++s) o[s] = make_float4(0.f, 0.f, 0.f, 0.f);
        const float top = fmaxf(warp_max(ml.x), sink2);
        const float w = ml.x == -INFINITY ? 0.0f : tc::exp2_approx(ml.x - top);
        float l = warp_sum(w * ml.y);
        if (a.sink) l += tc::exp2_approx(sink2 - top);
        for (int k = 0; k < it.parts; k += 2) {
            if (k) load(k);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float wk = __shfl_sync(0xffffffffu, w, k + j);       // 0 behind the last part
#pragma unroll
                for (int s = 0; s < 4; ++s) add_scaled(o[s], wk, x[j][s]);
            }
        }
        const float inv = l == 0.0f ? 0.0f : (1.0f / kLift) / l;
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s < slices) st_bf16x4(a.out + (it.row0 + row) * D + s * 128 + lane * 4, make_float4(o[s].x * inv, o[s].y * inv, o[s].z * inv, o[s].w * inv));
        if (lane == 0 && a.lse) a.lse[it.row0 + row] = lse_of(l, top, sink, sink2);
    }

    // SL slices of 128 dims in a CTA: all four where there are more rows than slices would leave CTAs for
    auto many = [&](auto sl) {
        constexpr int SL = decltype(sl)::value, kBatch = SL > 1 ? 2 : 6;
        const int cuts = slices / SL;
        for (int u = blockIdx.x; u < n_begun[1] * kRows * cuts; u += gridDim.x) {
            const int c = begun[1][u / (kRows * cuts)], row = u / cuts % kRows, slice = u % cuts * SL;
            const Meta &it = items[c];
            const int parts = it.parts;
            if (row >= it.rows) continue;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (tid < parts) ml = part_ml[part_of(c, tid) * kRows + row];
            const float sink = sink_of(it, row), sink2 = a.sink ? sink_log2(sink) : -INFINITY;
            float4 x[kBatch][SL], o[SL];
            auto load = [&](int k0) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int k = k0 + i * kJoinWarps;
                    const float4 *from = reinterpret_cast<const float4 *>(part_o + ((int64_t)part_of(c, k) * kRows + row) * D + slice * 128 + lane * 4);
#pragma unroll
                    for (int s = 0; s < SL; ++s) x[i][s] = k < parts ? ld_part(reinterpret_cast<const float *>(from + s * 32)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            };
            load(warp);
            const float warp_top = warp_max(ml.x);
            if (lane == 0) most_s[warp] = warp_top;
            __syncthreads();
            float top = sink2;
#pragma unroll
            for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, most_s[i]);
            const float w = ml.x == -INFINITY ? 0.0f : tc::exp2_approx(ml.x - top), warp_l = warp_sum(w * ml.y);
            if (tid < kCtas) weight[tid] = w;
            if (lane == 0) sum_s[warp] = warp_l;
            __syncthreads();
#pragma unroll
            for (int s = 0; s < SL; ++s) o[s] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int k0 = warp; k0 < parts; k0 += kBatch * kJoinWarps) {
                if (k0 != warp) load(k0);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const float wk = k0 + i * kJoinWarps < parts ? weight[k0 + i * kJoinWarps] : 0.0f;
#pragma unroll
                    for (int s = 0; s < SL; ++s) add_scaled(o[s], wk, x[i][s]);
                }
            }
#pragma unroll
            for (int s = 0; s < SL; ++s) sums[s][warp][lane] = o[s];
            __syncthreads();
            if (warp < SL) {
                float l = a.sink ? tc::exp2_approx(sink2 - top) : 0.0f;
#pragma unroll
                for (int i = 0; i < kJoinWarps; ++i) l += sum_s[i];
                float4 y = sums[warp][0][lane];
#pragma unroll
                for (int i = 1; i < kJoinWarps; ++i) add_scaled(y, 1.0f, sums[warp][i][lane]);
                const float inv = l == 0.0f ? 0.0f : (1.0f / kLift) / l;
                st_bf16x4(a.out + (it.row0 + row) * D + (slice + warp) * 128 + lane * 4, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                if (lane == 0 && slice + warp == 0 && a.lse) a.lse[it.row0 + row] = lse_of(l, top, sink, sink2);
            }
            __syncthreads();                             // sums and sum_s are read
        }
    };
    if (slices == 4 && n_begun[1] * kRows * slices > (int)gridDim.x) many(std::integral_constant<int, 4>());
    else many(std::integral_constant<int, 1>());
}

// The rows a chunk's tokens see, once each, as packed f16 rows: with a window of 128 rows every row is wanted by 128 tokens, and turning it into
// f16 for each of them cost more than all the rest (4096 tokens: 294 us straight from the cache).  One warp per row.
// A row of codes whose largest value is outside [2^-9, 2^15] is scaled by a power of two, its factor; f32 rows become f16 numbers as they
// do straight from the cache (beyond +-65504 that), so a token's rows do not depend on the path; a hole has the factor 0, a row with a value
// that is not finite NaN, with zeros in place of such values, so that it reaches the tokens that see it and no others.
template <int V>      // float4s of a row per lane: head_dim / 128
__global__ void __launch_bounds__(kPackWarps * 32) attn_pack_kernel(const AttnArgs a, int64_t bound, uint16_t *rows, float *fac, int *odd) {
    const int lane = threadIdx.x & 31, dim = a.kv.head_dim;
    const int64_t most = a.table_width * a.kv.page_rows, gap = packed_gap(a.window, a.n_first, most);
    bool met = false;
    launch_dependents();
    for (int64_t row = (int64_t)blockIdx.x * kPackWarps + (threadIdx.x >> 5); row < bound; row += (int64_t)kPackCtas * kPackWarps) {
        int lo = 0, hi = a.n_seqs - 1;                   // the last sequence that begins at or before this row
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (mid * gap + (a.window > 0 ? first_token(a, mid) - first_token(a, 0) : 0) <= row) lo = mid; else hi = mid - 1;
        }
        const Packed k = get_packed(a, lo);
        const int64_t local = row - k.off;
        if (local < 0 || local >= (int64_t)k.first + k.len - k.lo + 16) continue;      // 16 rows of zeros behind each sequence
        const bool is = local < (int64_t)k.first + k.len - k.lo;
        int64_t slot = -1;
        if (is) {
            const int at = local < k.first ? (int)local : (int)(local - k.first) + k.lo, pg = at / a.kv.page_rows;
            const int page = __ldg(a.page_table + lo * a.table_width + pg);
            if (page >= 0 && page < a.kv.n_pages) slot = (int64_t)page * a.kv.page_rows + (at - pg * a.kv.page_rows);
        }
        float4 r[V];
        float top = 0.0f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = 4 * (lane + 32 * j), nope = dim - a.kv.n_rot;
            r[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (slot >= 0) {
                if (a.kv.row_format == DS4B200_KV_F32) {
                    r[j] = ld_ro4(a.kv.raw + slot * dim + e);
                } else if (a.kv.row_format == DS4B200_KV_FP8_BLOCK64 && e >= nope) {
                    r[j] = ld_ro4(a.kv.tail + slot * a.kv.n_rot + (e - nope));
                } else {
                    const float sc = __ldg(a.kv.scales + (a.kv.row_format == DS4B200_KV_FP8_ROW ? slot : slot * (nope >> 6) + (e >> 6)));
                    uint32_t x, y;
                    e4m3x4(__ldg(reinterpret_cast<const uint32_t *>(a.kv.codes + slot * dim + e)), x, y);
                    const float2 f = f16x2_bits_to_f32(x), h = f16x2_bits_to_f32(y);
                    r[j] = make_float4(f.x * sc, f.y * sc, h.x * sc, h.y * sc);
                }
            }
            finite = finite && amax4(r[j]) < INFINITY && r[j].x == r[j].x && r[j].y == r[j].y && r[j].z == r[j].z && r[j].w == r[j].w;
            top = fmaxf(top, amax4(r[j]));
        }
        float f = !is || slot >= 0 ? 1.0f : 0.0f, down = 1.0f;
        if (!__all_sync(0xffffffffu, finite)) {
            f = __uint_as_float(0x7fffffffu);
#pragma unroll
            for (int j = 0; j < V; ++j) r[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
            top = warp_max(top);
            if (a.kv.row_format != DS4B200_KV_F32 && top != 0.0f && (top < 0x1p-9f || top > 0x1p15f)) pow2_parts(fmaxf(top, kLeast), f, down);
        }
        met = met || f != 1.0f;
        if (lane == 0) fac[row] = f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint2 u = make_uint2(sat_h2(r[j].x * down, r[j].y * down), sat_h2(r[j].z * down, r[j].w * down));
            *reinterpret_cast<uint2 *>(rows + row * dim + 4 * (lane + 32 * j)) = u;
        }
    }
    met = __syncthreads_or(met);
    if (threadIdx.x == 0) odd[blockIdx.x] = met;
}

bool packed_map(CUtensorMap *map, const uint16_t *rows, int64_t n, int dim, int box_rows) {
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            encode = reinterpret_cast<EncodeFn>(fn);
        else
            cudaGetLastError();
    });
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)n}, strides[1] = {(cuuint64_t)dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<uint16_t *>(rows), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The workspace holds either the parts of cut items or packed rows.
constexpr int64_t kPackRows = 4 * kCtas * kRows;         // f16 rows in the room of 2 kCtas kRows f32 ones
constexpr int64_t kMetaBytes = (kCtas * (int64_t)sizeof(Meta) + 127) / 128 * 128;
constexpr int64_t kMlBytes = 2 * kCtas * kRows * (int64_t)sizeof(float2);

template <int NB, int FMT, bool SHARED>
bool launch_tc(const TcArgs &g, cudaStream_t s) {
    constexpr int kSmem = 3 * kRows * NB * 256 + (FMT == kPacked ? 3 : 2) * 8192;
    constexpr int kOneCta = 120 * 1024;               // one CTA per SM: each takes the whole tensor memory
    const int smem = kSmem > kOneCta ? kSmem : kOneCta;
    const auto kernel = attn_tc_kernel<NB, FMT, SHARED>;
    static const bool enough = [&] {                 // a compiler that gives the kernel fewer registers than the roles' split needs
        cudaFuncAttributes at;
        return cudaFuncGetAttributes(&at, kernel) == cudaSuccess && at.numRegs >= kLaunchRegs;
    }();
    if (!enough || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
    const unsigned grid = (unsigned)(g.split || g.n_slots > kCtas ? kCtas : g.n_slots);
    if (FMT == kPacked) launch_behind(kernel, grid, kThreads, smem, s, g);
    else kernel<<<grid, kThreads, smem, s>>>(g);
    if (g.split) launch_behind(attn_join_kernel, kJoinCtas, kJoinWarps * 32, 0, s, g.a, (const Meta *)g.meta, (const float2 *)g.part_ml, (const float *)g.part_o);
    return true;
}

template <int NB>
bool launch_fmt(const AttnArgs &a, cudaStream_t s) {
    TcArgs g{};
    g.a = a;
    g.head_groups = (a.n_heads + kRows - 1) / kRows;
    g.group = a.q_start && g.head_groups == 1 ? kRows / a.n_heads : 1;
    const int64_t slots = (a.q_start ? a.n_tokens / g.group + a.n_seqs + 1 : a.n_seqs) * g.head_groups;
    g.n_slots = (int)slots;
    // Equal runs of tiles pay where items are long and few: a run's two ends cost 128 KiB of partial sums each and the join another launch.
    // The host knows the table's width and not the lengths, so the width stands for them: 592 sequences of 120 rows take 46 us under a table
    // of two pages and 50, cut, under one of 1000.  Tiles: 512 prompt tokens of 3 tiles take 30 us as whole items and 79 cut (512 dims, replayed).
    // Items: a chunk's are many and alike, and cutting them costs (1000 tokens of 128 dims, window 512: 42 us whole, 110 cut; nine prompts
    // of 1531 tokens 76 and 182).  A decode's gain little from it where they are alike (592 sequences of 2000 rows 255 us whole, 259 cut; 1200 of
    // 1000 rows 296 and 314) and much where they are not (592 of up to 8000 rows 771 and 491; 591 of 1000 rows beside one of 65536
    // 1834 and 190), also beyond kSplitItems, where they are whole all the same (600 of up to 8000 rows: 771, cut they would take 494).
    const int64_t all_rows = a.table_width * a.kv.page_rows;
    const int64_t seen = a.window > 0 ? std::min<int64_t>(all_rows, (int64_t)a.window + a.n_first + g.group - 1) : all_rows;
    g.split = seen > kWholeTiles * kRows && slots <= kSplitItems;
    g.page_shift = -1;
    for (int k = 0; k < 31; ++k) if (a.kv.page_rows == 1 << k) g.page_shift = k;
    unsigned char *ws = static_cast<unsigned char *>(a.ws);
    g.meta = reinterpret_cast<Meta *>(ws);
    g.part_ml = reinterpret_cast<float2 *>(ws + kMetaBytes);
    g.part_o = reinterpret_cast<float *>(ws + kMetaBytes + kMlBytes);
    g.status = device_status_word();
    static_assert(kPackCtas * sizeof(int) <= kMetaBytes && kPackRows * sizeof(float) <= kMlBytes && kPackCtas <= kThreads, "room for packed rows");
    const int64_t bound = (a.window > 0 ? a.n_tokens : 0) + a.n_seqs * packed_gap(a.window, a.n_first, all_rows);
    uint16_t *rows = reinterpret_cast<uint16_t *>(g.part_o);
    // Packing pays where a row is wanted by more than one item of a CTA, and where tokens share an item (masks straight from the cache
    // cost more than the launch): 256 tokens of 64 heads 37 us straight, 27 packed, 128 tokens 20.4 and 22.5; of 8 heads, 32 tokens
    // 27 and 20, 128 tokens 27 and 20.  (Window 128, 4 first rows.)
    if (a.q_start && !g.split && (g.group > 1 || slots > kCtas) && bound <= kPackRows && packed_map(&g.rows, rows, bound, a.kv.head_dim, 64) &&
        packed_map(&g.few, rows, bound, a.kv.head_dim, 16)) {
        g.fac = reinterpret_cast<const float *>(g.part_ml);
        g.odd = reinterpret_cast<const int *>(ws);
        attn_pack_kernel<NB><<<kPackCtas, kPackWarps * 32, 0, s>>>(a, bound, rows, reinterpret_cast<float *>(g.part_ml), reinterpret_cast<int *>(ws));
        return launch_tc<NB, kPacked, true>(g, s);
    }
    switch (a.kv.row_format) {
        case DS4B200_KV_F32: return g.group > 1 ? launch_tc<NB, DS4B200_KV_F32, true>(g, s) : launch_tc<NB, DS4B200_KV_F32, false>(g, s);
        case DS4B200_KV_FP8_ROW: return g.group > 1 ? launch_tc<NB, DS4B200_KV_FP8_ROW, true>(g, s) : launch_tc<NB, DS4B200_KV_FP8_ROW, false>(g, s);
        default: return g.group > 1 ? launch_tc<NB, DS4B200_KV_FP8_BLOCK64, true>(g, s) : launch_tc<NB, DS4B200_KV_FP8_BLOCK64, false>(g, s);
    }
}

}  // namespace

int64_t attn_workspace_bytes(int n_heads, int head_dim) {
    return kMetaBytes + kMlBytes + 2 * kCtas * kRows * (int64_t)head_dim * 4;
}

bool attn_paged(const AttnArgs &a, cudaStream_t s) {
    switch (a.kv.head_dim / 128) {
        case 1: return launch_fmt<1>(a, s);
        case 2: return launch_fmt<2>(a, s);
        case 3: return launch_fmt<3>(a, s);
        default: return launch_fmt<4>(a, s);
    }
}

}  // namespace ds4b200
