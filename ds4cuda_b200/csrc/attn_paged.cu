// attn_paged.cu — attention over a paged key-value cache: one new token per sequence, or the tokens of a
// prompt chunk with a sliding window and first rows that stay visible.
//
// Mathematics: o_h = sum_j exp(s_hj - lse_h) k_j with s_hj = scale q_h . k_j over the visible rows j and
// lse_h = log(sum_j exp(s_hj) + exp(sink_h)).  One row is key and value of every head (the reference's
// cache has one KV head; cuda/flash_attn.cu:148-313).
#include <mutex>

#include "device_utils.cuh"
#include "kernels.cuh"
#include "tcgen05_utils.cuh"

namespace ds4b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------------------------- tensor cores
//
// An item is up to 64 query rows that share their cache rows: the heads of one token (of up to 64 / n_heads tokens,
// when a chunk's heads are few).  A CTA walks over tiles of 64 cache rows:
//   * eight warps load the tile's rows through the page table, turn them into f16 and store them once, as 128-byte
//     rows of 64 dims with the 128-byte swizzle.  The same bytes serve both products: as the K-major B operand of
//     S = Q K^T and as the M-contiguous A operand of O^T += V^T P^T, since a key row is its value row;
//   * one thread issues the MMAs: S (M 64 query rows, N 64 cache rows, K head_dim) and, per 128 dims of the output,
//     O^T (M 128 dims, N query rows, K 64 cache rows).  O^T takes 64 tensor-memory columns per 128 dims, so 512 dims and two S
//     buffers fit; O itself (64 rows in 512 columns) would leave no room for S;
//   * four warps take S from tensor memory, one query row per lane, keep the running maximum and sum of the softmax in f32,
//     and leave the weights as f16 (relative error 2^-12) in shared memory.  The accumulators are rescaled only when a
//     row's maximum has grown by more than 2^8 since its last reference, which later tiles rarely bring.
// S of tile n + 1 is issued ahead of O^T of tile n, so the tensor cores work while the softmax of a tile runs.
//
// Scales.  A cache row is a row factor times f16 numbers: E4M3 codes themselves with the row's scale; codes times their
// block's scale relative to the row's largest power of two (exact, the scales are powers of two) with the f32 tail likewise; f32 rows as they are.
// The factor r_j enters the scores, and as log2 r_j the exponent of the weights, so that P holds r_j exp(s_j - M) <= 1
// and the sum takes P / r_j back.  A query row is scaled by a power of two, which loses nothing of bf16's 8 bits in f16.
//
// Work.  With few items the list of all tiles is cut into equal runs, one per CTA; an item that several CTAs share leaves
// partial sums (f32 O^T, M and l) that attn_join_kernel adds in order.  With many items each CTA takes whole ones.
constexpr int kCtas = 148;
constexpr int kRows = 64;                   // query rows of an item, cache rows of a tile
constexpr int kLoadWarp0 = 4, kLoadWarps = 8, kMmaWarp = 12;
constexpr int kThreads = 13 * 32;
constexpr int kSplitItems = 4 * kThreads;   // up to this many items the tiles are cut into equal runs
constexpr int kMinTiles = 2;                // of a run: below, the join costs more than the run saves
constexpr float kRescale = 8.0f;            // log2 units
constexpr int kScaleSets = 4;

struct Meta { int64_t row0; int rows, parts; };

struct Item {
    int64_t row0;                           // first row of q / out, n_heads rows per token
    int b, rows, p0, first, lo, n, tiles;
};

__device__ __forceinline__ Item get_item(const AttnArgs &a, int group, int head_groups, int slot) {
    Item it;
    const int g = slot / head_groups, hg = slot - g * head_groups;
    int tok0, ntok = 1;
    if (a.q_start) {
        // sequence b's groups take the slots from q_start[b] / group + b on (one slot per sequence may stay empty)
        int lo = 0, hi = a.n_seqs - 1;
        const int off = a.q_start[0] / group;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.q_start[mid] / group + mid - off <= g) lo = mid; else hi = mid - 1;
        }
        it.b = lo;
        const int q0 = a.q_start[lo], q1 = a.q_start[lo + 1];
        const int local = (g - (q0 / group + lo - off)) * group;
        tok0 = q0 + local;
        ntok = min(group, (int)min((int64_t)q1, a.n_tokens) - tok0);
        if (tok0 < 0) ntok = 0;
        it.p0 = local - (q1 - q0);
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
    it.tiles = ntok <= 0 ? 0 : max(1, (it.n + kRows - 1) / kRows);
    it.row0 = (int64_t)tok0 * a.n_heads + hg * kRows;
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

// A CTA's run: segments of items.  next() gives the coming segment's item and its tiles [t0, t1).
struct Walk {
    int slot, tile, step;
    long long left;
    __device__ __forceinline__ bool next(const AttnArgs &a, int group, int head_groups, int n_slots, Item &it, int &t0, int &t1) {
        while (left > 0 && slot < n_slots) {
            it = get_item(a, group, head_groups, slot);
            slot += step;
            if (it.tiles == 0) continue;
            t0 = tile;
            t1 = (int)min((long long)it.tiles, t0 + left);
            tile = 0;
            if (step == 1) left -= t1 - t0;
            return true;
        }
        return false;
    }
};

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 e4m3x2(uint32_t two) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3));
}
__device__ __forceinline__ uint32_t sat_h2(float x, float y) {      // finite values beyond f16 become +-65504
    x = fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
    y = fabsf(y) < INFINITY ? fminf(fmaxf(y, -65504.f), 65504.f) : y;
    return h2_bits(__floats2half2_rn(x, y));
}
// 2^e and 2^-e with e the exponent of x (0 for x = 0), both normal
__device__ __forceinline__ void pow2_parts(float x, float &up, float &down) {
    int e = (int)((__float_as_uint(x) >> 23) & 255u) - 127;
    if (x == 0.0f) e = 0;
    e = min(max(e, -126), 126);
    up = __uint_as_float((uint32_t)(e + 127) << 23);
    down = __uint_as_float((uint32_t)(127 - e) << 23);
}

template <int NB, int FMT>          // NB: head_dim / 128
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const AttnArgs a, int group, int head_groups, int n_slots, int split,
                                                              Meta *meta, float2 *part_ml, float *part_o, int *status) {
    constexpr int D = NB * 128, kChunks = NB * 2, kTileBytes = kRows * D * 2;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char *q_s = smem, *k_s = smem + kTileBytes, *p_s = smem + 3 * kTileBytes;
    __shared__ __align__(8) uint64_t full[2], s_full[2], s_free[2], p_full[2], pv_done[2], q_full, q_free;
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s, start_slot, start_tile;
    __shared__ long long scan_s[kThreads / 32];
    __shared__ __align__(16) float row_mul[2][kRows], row_add[2][kRows], row_div[2][kRows];
    __shared__ __align__(16) int row_at[2][kRows];
    __shared__ float q_mul[kScaleSets][kRows];
    __shared__ __align__(16) float fac_s[kRows], inv_s[kRows];
    volatile int *abort_flag = &abort_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        abort_s = 0;
        start_slot = n_slots;
        start_tile = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], kLoadWarps); mbar_init(&s_full[i], 1); mbar_init(&s_free[i], 4);
            mbar_init(&p_full[i], 4); mbar_init(&pv_done[i], 1);
        }
        mbar_init(&q_full, kLoadWarps); mbar_init(&q_free, 1);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_s)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    Walk start{(int)blockIdx.x, 0, (int)gridDim.x, 1ll << 62};
    long long per = 0, total = 0;
    if (split) {
        for (int base = 0; base < n_slots; base += kThreads) {
            const int s = base + tid;
            long long sum;
            block_scan64(s < n_slots ? get_item(a, group, head_groups, s).tiles : 0, scan_s, &sum);
            total += sum;
        }
        per = max((long long)kMinTiles, (total + kCtas - 1) / kCtas);
        const long long from = per * blockIdx.x;
        long long seen = 0;
        for (int base = 0; base < n_slots; base += kThreads) {
            const int s = base + tid;
            const int tiles = s < n_slots ? get_item(a, group, head_groups, s).tiles : 0;
            long long sum;
            const long long before = seen + block_scan64(tiles, scan_s, &sum);
            if (before <= from && from < before + tiles) { start_slot = s; start_tile = (int)(from - before); }
            seen += sum;
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_s, s_tmem = tmem + NB * 64;
    if (split) start = Walk{start_slot, start_tile, 1, min(per, total - per * (long long)blockIdx.x)};

    if (warp >= kLoadWarp0 && warp < kLoadWarp0 + kLoadWarps) {
        // ------------------------------------------------------------------------------ loaders
        const int r = (warp - kLoadWarp0) * 8 + (lane >> 2), part = lane & 3;   // four lanes per row, 16 of 64 dims each
        const uint32_t row_off = (uint32_t)(r * 128), sw = (uint32_t)(r & 7);
        const bool tail = FMT == DS4B200_KV_FP8_BLOCK64 && a.kv.n_rot != 0;
        const int n_scales = FMT == DS4B200_KV_FP8_BLOCK64 ? (D - a.kv.n_rot) / 64 : 1;
        Walk w = start;
        Item it;
        int t0, t1, n = 0, seg = 0;
        while (w.next(a, group, head_groups, n_slots, it, t0, t1)) {
            const int32_t *table = a.page_table + it.b * a.table_width;
            int at = 0;
            auto find = [&](int t) -> int64_t {          // slot of this lane's row of tile t, or -1
                const int i = t * kRows + r;
                at = i < it.first ? i : it.lo + (i - it.first);
                if (i >= it.n) return -1;
                const int pg = at / a.kv.page_rows;
                const int page = __ldg(table + pg);
                return page < 0 || page >= a.kv.n_pages ? -1 : (int64_t)page * a.kv.page_rows + (at - pg * a.kv.page_rows);
            };
            int64_t slot = find(t0);
            {   // the item's query rows
                uint4 v[kChunks][2];
                uint32_t amax = 0;
                const uint16_t *src = a.q + (it.row0 + r) * D + part * 16;
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        v[c][u] = r < it.rows ? __ldg(reinterpret_cast<const uint4 *>(src + c * 64 + u * 8)) : make_uint4(0, 0, 0, 0);
                        const uint32_t x[4] = {v[c][u].x, v[c][u].y, v[c][u].z, v[c][u].w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) amax = max(amax, max(x[k] & 0x7fff0000u, (x[k] << 16) & 0x7fff0000u));
                    }
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                float up, down;
                pow2_parts(__uint_as_float(amax), up, down);
                tc::wait(&q_free, (uint32_t)((seg & 1) ^ 1), abort_flag, status);
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t x[4] = {v[c][u].x, v[c][u].y, v[c][u].z, v[c][u].w};
                        uint32_t o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            o[k] = h2_bits(__floats2half2_rn(__uint_as_float(x[k] << 16) * down, __uint_as_float(x[k] & 0xffff0000u) * down));
                        *reinterpret_cast<uint4 *>(q_s + c * 8192 + row_off + (((uint32_t)(part * 2 + u) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                if (part == 0) q_mul[seg & (kScaleSets - 1)][r] = up * a.scale * kLog2e;
                tc::fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
            for (int t = t0; t < t1; ++t, ++n) {
                const int buf = n & 1;
                unsigned char *dst = k_s + buf * kTileBytes + row_off;
                const uint32_t use = (uint32_t)(((n >> 1) & 1) ^ 1);
                const int64_t my = slot;
                const int my_at = at;
                float mul = 1.0f;
                if (FMT == DS4B200_KV_F32) {
                    constexpr int kHalf = kChunks > 4 ? 4 : kChunks;
                    const float *src = a.kv.raw + my * D + part * 4;
#pragma unroll
                    for (int h = 0; h < kChunks; h += kHalf) {
                        float4 v[kHalf][4];
#pragma unroll
                        for (int c = 0; c < kHalf; ++c)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (h + c < kChunks)
                                    v[c][j] = my >= 0 ? __ldg(reinterpret_cast<const float4 *>(src + (h + c) * 64 + j * 16)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        if (h == 0) {
                            slot = t + 1 < t1 ? find(t + 1) : -1;
                            tc::wait(&pv_done[buf], use, abort_flag, status);
                        }
#pragma unroll
                        for (int c = 0; c < kHalf; ++c)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (h + c < kChunks)
                                    *reinterpret_cast<uint2 *>(dst + (h + c) * 8192 + (((uint32_t)(2 * j + (part >> 1)) ^ sw) << 4) + (part & 1) * 8) =
                                        make_uint2(sat_h2(v[c][j].x, v[c][j].y), sat_h2(v[c][j].z, v[c][j].w));
                    }
                } else {
                    uint4 v[kChunks];
                    float4 tl[4];
                    float sc0 = 0.0f, sc1 = 0.0f;
                    const uint8_t *src = a.kv.codes + my * D + part * 16;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        v[c] = my >= 0 && !(tail && c == kChunks - 1) ? __ldg(reinterpret_cast<const uint4 *>(src + c * 64)) : make_uint4(0, 0, 0, 0);
                    if (FMT == DS4B200_KV_FP8_ROW) {
                        if (my >= 0) mul = __ldg(a.kv.scales + my);
                    } else {
                        if (my >= 0 && part < n_scales) sc0 = __ldg(a.kv.scales + my * n_scales + part);
                        if (my >= 0 && part + 4 < n_scales) sc1 = __ldg(a.kv.scales + my * n_scales + part + 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tl[j] = my >= 0 && tail ? __ldg(reinterpret_cast<const float4 *>(a.kv.tail + my * 64 + part * 16 + j * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    slot = t + 1 < t1 ? find(t + 1) : -1;
                    float down = 1.0f;
                    if (FMT == DS4B200_KV_FP8_BLOCK64) {
                        float top = fmaxf(fmaxf(amax4(tl[0]), amax4(tl[1])), fmaxf(amax4(tl[2]), amax4(tl[3]))) * (1.0f / 256.0f);
                        top = fmaxf(top, fmaxf(sc0, sc1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        pow2_parts(top, mul, down);
                        sc0 *= down;
                        sc1 *= down;
                    }
                    tc::wait(&pv_done[buf], use, abort_flag, status);
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        uint32_t o[8];
                        const uint32_t x[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            o[2 * k] = h2_bits(e4m3x2(x[k] & 0xffffu));
                            o[2 * k + 1] = h2_bits(e4m3x2(x[k] >> 16));
                        }
                        if (FMT == DS4B200_KV_FP8_BLOCK64) {
                            const __half2 f = __float2half2_rn(__shfl_sync(0xffffffffu, c < 4 ? sc0 : sc1, (lane & ~3) | (c & 3)));
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = h2_bits(__hmul2(*reinterpret_cast<__half2 *>(&o[k]), f));
                            if (tail && c == kChunks - 1) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    o[2 * j] = h2_bits(__floats2half2_rn(tl[j].x * down, tl[j].y * down));
                                    o[2 * j + 1] = h2_bits(__floats2half2_rn(tl[j].z * down, tl[j].w * down));
                                }
                            }
                        }
                        *reinterpret_cast<uint4 *>(dst + c * 8192 + (((uint32_t)(part * 2) ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4 *>(dst + c * 8192 + (((uint32_t)(part * 2 + 1) ^ sw) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                    }
                }
                if (part == 0) {
                    mul = mul == 0.0f ? 1.0e-30f : mul;
                    if (FMT != DS4B200_KV_F32) { row_mul[buf][r] = mul; row_div[buf][r] = 1.0f / mul; }
                    row_add[buf][r] = my >= 0 ? (FMT == DS4B200_KV_F32 ? 0.0f : log2f(mul)) : -INFINITY;
                    row_at[buf][r] = my_at;
                }
                tc::fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[buf]);
            }
            ++seg;
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            const uint64_t q_desc = tc::desc(smem_addr(q_s), 0), k_desc = tc::desc(smem_addr(k_s), 0);
            const uint64_t v_desc = tc::desc(smem_addr(k_s), 8192), p_desc = tc::desc(smem_addr(p_s), 0);
            constexpr uint32_t s_idesc = tc::idesc_f16(64, 64, false);
            auto weighted = [&](int k, bool fresh, uint32_t o_idesc) {      // O^T (+)= V^T P^T of tile k
                const int buf = k & 1;
                tc::wait(&p_full[buf], (uint32_t)((k >> 1) & 1), abort_flag, status);
                tc::fence_after();
#pragma unroll
                for (int m = 0; m < NB; ++m)
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        tc::mma_f16(tmem + m * 64, v_desc + (uint64_t)((buf * kTileBytes + m * 16384 + ks * 2048) >> 4),
                                    p_desc + (uint64_t)((buf * 8192 + ks * 32) >> 4), o_idesc, !(fresh && ks == 0));
                tc::commit(&pv_done[buf]);
            };
            Walk w = start;
            Item it;
            int t0, t1, n = 0, seg = 0;
            bool fresh = false;
            uint32_t o_idesc = 0;
            while (w.next(a, group, head_groups, n_slots, it, t0, t1)) {
                tc::wait(&q_full, (uint32_t)(seg & 1), abort_flag, status);
                for (int t = t0; t < t1; ++t, ++n) {
                    const int buf = n & 1;
                    tc::wait(&full[buf], (uint32_t)((n >> 1) & 1), abort_flag, status);
                    tc::wait(&s_free[buf], (uint32_t)(((n >> 1) & 1) ^ 1), abort_flag, status);
                    tc::fence_after();
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            tc::mma_f16(s_tmem + buf * 64, q_desc + (uint64_t)((c * 8192 + ks * 32) >> 4),
                                        k_desc + (uint64_t)((buf * kTileBytes + c * 8192 + ks * 32) >> 4), s_idesc, c > 0 || ks > 0);
                    tc::commit(&s_full[buf]);
                    if (t + 1 == t1) tc::commit(&q_free);
                    if (n > 0) weighted(n - 1, fresh, o_idesc);
                    fresh = t == t0;
                    o_idesc = tc::idesc_f16(128, (it.rows + 15) / 16 * 16, true);
                }
                ++seg;
            }
            if (n > 0) weighted(n - 1, fresh, o_idesc);
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------------------ softmax and output
        const int row = warp * 16 + lane;               // lanes 0-15 hold a row of S each
        const bool mine = lane < 16;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const bool several = head_groups == 1 && group > 1;
        Meta last{0, 0, 0};
        Walk w = start;
        Item it;
        int t0, t1, n = 0, seg = 0;
        long long done = 0;
        while (w.next(a, group, head_groups, n_slots, it, t0, t1)) {
            float qk = 0.0f;
            const int p = it.p0 + (several ? (row & 63) / a.n_heads : 0);
            const int from = a.window > 0 ? p - a.window : -1;      // rows above it are in the window
            float m = -INFINITY, l = 0.0f;
            for (int t = t0; t < t1; ++t, ++n) {
                const int buf = n & 1;
                tc::wait(&full[buf], (uint32_t)((n >> 1) & 1), abort_flag, status);
                tc::wait(&s_full[buf], (uint32_t)((n >> 1) & 1), abort_flag, status);
                tc::fence_after();
                // written ahead of the segment's first tile by the same warps; q_full itself may be phases ahead of this warp
                if (t == t0 && mine) qk = q_mul[seg & (kScaleSets - 1)][row];
                uint32_t x0[32], x1[32];
                tc::ld32(s_tmem + buf * 64 + lane_base, x0);
                tc::ld32(s_tmem + buf * 64 + 32 + lane_base, x1);
                tc::wait_ld();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[buf]);
                float v[64];
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 64; j += 4) {
                    const float4 add = *reinterpret_cast<const float4 *>(&row_add[buf][j]);
                    const float ad[4] = {add.x, add.y, add.z, add.w};
                    float mu[4] = {1.f, 1.f, 1.f, 1.f};
                    if (FMT != DS4B200_KV_F32) {
                        const float4 f = *reinterpret_cast<const float4 *>(&row_mul[buf][j]);
                        mu[0] = f.x; mu[1] = f.y; mu[2] = f.z; mu[3] = f.w;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float s = __uint_as_float(j + k < 32 ? x0[(j + k) & 31] : x1[(j + k) & 31]) * qk;
                        v[j + k] = fmaf(s, mu[k], ad[k]);
                    }
                    if (several) {
                        const int4 at4 = *reinterpret_cast<const int4 *>(&row_at[buf][j]);
                        const int at[4] = {at4.x, at4.y, at4.z, at4.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (at[k] > p || (at[k] <= from && at[k] >= a.n_first)) v[j + k] = -INFINITY;
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) top = fmaxf(top, v[j + k]);
                }
                const bool grown = mine && m > -INFINITY && top > m + kRescale;
                uint32_t any;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                             : "=r"(any) : "r"((uint32_t)grown) : "memory");
                if (any) {
                    // every row's accumulators (a column of O^T) follow its maximum; the previous tile's MMAs first
                    const float f = grown ? exp2f(m - top) : 1.0f;
                    if (grown) { m = top; l *= f; }
                    if (mine) fac_s[row] = f;
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    if (t > t0) {
                        tc::wait(&pv_done[buf ^ 1], (uint32_t)(((n - 1) >> 1) & 1), abort_flag, status);
                        tc::fence_after();
                        for (int col = 0; col < (it.rows + 15) / 16 * 16; col += 16)
#pragma unroll 1
                            for (int b = 0; b < NB; ++b) {
                                uint32_t o[16];
                                tc::ld16(tmem + b * 64 + col + lane_base, o);
                                tc::wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * fac_s[col + k]);
                                tc::st16(tmem + b * 64 + col + lane_base, o);
                            }
                        tc::wait_st();
                    }
                }
                if (m == -INFINITY) m = top;
                const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int j = 0; j < 64; j += 8) {
                    uint32_t o[4];
#pragma unroll
                    for (int k = 0; k < 8; k += 4) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) e[i] = exp2f(v[j + k + i] - ref);
                        if (FMT == DS4B200_KV_F32) {
                            l += (e[0] + e[1]) + (e[2] + e[3]);
                        } else {
                            const float4 d = *reinterpret_cast<const float4 *>(&row_div[buf][j + k]);
                            l += fmaf(e[0], d.x, e[1] * d.y) + fmaf(e[2], d.z, e[3] * d.w);
                        }
                        o[k / 2] = h2_bits(__floats2half2_rn(e[0], e[1]));
                        o[k / 2 + 1] = h2_bits(__floats2half2_rn(e[2], e[3]));
                    }
                    if (mine)
                        *reinterpret_cast<uint4 *>(p_s + buf * 8192 + row * 128 + (((uint32_t)(j / 8) ^ (uint32_t)(row & 7)) << 4)) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                }
                tc::fence_async();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[buf]);
            }
            // the segment's accumulators
            tc::wait(&pv_done[(n - 1) & 1], (uint32_t)(((n - 1) >> 1) & 1), abort_flag, status);
            tc::fence_after();
            const bool whole = t0 == 0 && t1 == it.tiles;
            float inv = 1.0f;
            const int part = 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0);
            if (whole) {
                const float mine2 = l > 0.0f ? m + log2f(l) : (l == l ? -INFINITY : l);
                float lse2 = mine2;
                if (a.sink && mine && row < it.rows) {
                    const float s2 = a.sink[(it.row0 + row) % a.n_heads] * kLog2e, hi = fmaxf(mine2, s2);
                    lse2 = hi == -INFINITY ? hi : hi + log2f(exp2f(mine2 - hi) + exp2f(s2 - hi));
                }
                inv = m == -INFINITY ? 0.0f : exp2f(m - lse2);
                if (a.lse && mine && row < it.rows) a.lse[it.row0 + row] = lse2 * (1.0f / kLog2e);
            } else if (mine) {
                part_ml[part * kRows + row] = make_float2(m, l);
            }
            if (mine) inv_s[row] = inv;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int b = 0; b < NB; ++b)
                for (int col = 0; col < it.rows; col += 16) {
                    uint32_t o[16];
                    tc::ld16(tmem + b * 64 + col + lane_base, o);
                    tc::wait_ld();
                    const int d = b * 128 + warp * 32 + lane;
                    if (whole) {
                        uint16_t *dst = a.out + (it.row0 + col) * D + d;
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (col + k < it.rows) dst[k * D] = bf16_bits(__uint_as_float(o[k]) * inv_s[col + k]);
                    } else {
                        float *dst = part_o + ((int64_t)part * kRows + col) * D + d;
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (col + k < it.rows) dst[k * D] = __uint_as_float(o[k]);
                    }
                }
            tc::fence_before();
            if (t0 == 0 && t1 < it.tiles)
                last = Meta{it.row0, it.rows, (int)((per * (long long)blockIdx.x + done + it.tiles - 1) / per) - (int)blockIdx.x + 1};
            done += t1 - t0;
            ++seg;
        }
        if (split && tid == 0) meta[blockIdx.x] = last;
    }
    tc::fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Joins the parts of the item that CTA blockIdx.x began and did not finish; one query row per CTA.
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a, const Meta *meta, const float2 *part_ml, const float *part_o) {
    __shared__ float weight[kCtas];
    __shared__ float red[8];
    const Meta it = meta[blockIdx.x];
    const int row = blockIdx.y, D = a.kv.head_dim, tid = threadIdx.x;
    if (row >= it.rows || it.parts < 2) return;
    auto part_of = [&](int k) { return k == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + k); };
    const float sink2 = a.sink ? a.sink[(it.row0 + row) % a.n_heads] * kLog2e : -INFINITY;
    float hi = sink2;
    for (int k = tid; k < it.parts; k += 128) {
        const float2 ml = part_ml[part_of(k) * kRows + row];
        const float v = ml.y > 0.0f ? ml.x + log2f(ml.y) : (ml.y == ml.y ? -INFINITY : ml.y);
        weight[k] = v;
        hi = fmaxf(hi, v);
    }
    hi = warp_max(hi);
    if ((tid & 31) == 0) red[tid >> 5] = hi;
    __syncthreads();
    hi = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float sum = 0.0f;
    for (int k = tid; k < it.parts; k += 128) sum += hi == -INFINITY ? 0.0f : exp2f(weight[k] - hi);
    sum = warp_sum(sum);
    if ((tid & 31) == 0) red[4 + (tid >> 5)] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    if (a.sink && hi > -INFINITY) sum += exp2f(sink2 - hi);
    const float lse2 = hi == -INFINITY ? hi : hi + log2f(sum);
    __syncthreads();
    for (int k = tid; k < it.parts; k += 128) {
        const float m = part_ml[part_of(k) * kRows + row].x;
        weight[k] = m == -INFINITY ? 0.0f : exp2f(m - lse2);
    }
    __syncthreads();
    if (tid == 0 && a.lse) a.lse[it.row0 + row] = lse2 * (1.0f / kLog2e);
    if (4 * tid < D) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < it.parts; ++k) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(part_o + ((int64_t)part_of(k) * kRows + row) * D + 4 * tid));
            const float w = weight[k];
            o = make_float4(fmaf(w, v.x, o.x), fmaf(w, v.y, o.y), fmaf(w, v.z, o.z), fmaf(w, v.w, o.w));
        }
        st_bf16x4(a.out + (it.row0 + row) * D + 4 * tid, o);
    }
}

constexpr int64_t kMetaBytes = (kCtas * (int64_t)sizeof(Meta) + 127) / 128 * 128;
constexpr int64_t kMlBytes = 2 * kCtas * kRows * (int64_t)sizeof(float2);

template <int NB, int FMT>
void launch_tc(const AttnArgs &a, cudaStream_t s) {
    const int head_groups = (a.n_heads + kRows - 1) / kRows;
    const int group = a.q_start && head_groups == 1 ? kRows / a.n_heads : 1;
    const int64_t slots = (a.q_start ? a.n_tokens / group + a.n_seqs + 1 : a.n_seqs) * head_groups;
    const int split = slots <= kSplitItems;
    unsigned char *ws = static_cast<unsigned char *>(a.ws);
    Meta *meta = reinterpret_cast<Meta *>(ws);
    float2 *ml = reinterpret_cast<float2 *>(ws + kMetaBytes);
    float *po = reinterpret_cast<float *>(ws + kMetaBytes + kMlBytes);
    constexpr int kSmem = 3 * kRows * NB * 256 + 2 * 8192;
    constexpr int kOneCta = 120 * 1024;               // one CTA per SM: each takes the whole tensor memory
    const int smem = kSmem > kOneCta ? kSmem : kOneCta;
    static std::once_flag once[16];
    int dev = 0;
    cudaGetDevice(&dev);
    std::call_once(once[dev & 15], [&] { cudaFuncSetAttribute(attn_tc_kernel<NB, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    const unsigned grid = (unsigned)(split || slots > kCtas ? kCtas : slots);
    attn_tc_kernel<NB, FMT><<<grid, kThreads, smem, s>>>(a, group, head_groups, (int)slots, split, meta, ml, po, device_status_word());
    if (split) attn_join_kernel<<<dim3(kCtas, kRows), 128, 0, s>>>(a, meta, ml, po);
}

template <int NB>
void launch_fmt(const AttnArgs &a, cudaStream_t s) {
    if (a.kv.row_format == DS4B200_KV_F32) launch_tc<NB, DS4B200_KV_F32>(a, s);
    else if (a.kv.row_format == DS4B200_KV_FP8_ROW) launch_tc<NB, DS4B200_KV_FP8_ROW>(a, s);
    else launch_tc<NB, DS4B200_KV_FP8_BLOCK64>(a, s);
}

}  // namespace

int64_t attn_workspace_bytes(int n_heads, int head_dim) {
    return kMetaBytes + kMlBytes + 2 * kCtas * kRows * (int64_t)head_dim * 4;
}

void attn_paged(const AttnArgs &a, cudaStream_t s) {
    switch (a.kv.head_dim / 128) {
        case 1: launch_fmt<1>(a, s); break;
        case 2: launch_fmt<2>(a, s); break;
        case 3: launch_fmt<3>(a, s); break;
        default: launch_fmt<4>(a, s); break;
    }
}

}  // namespace ds4b200
