// attn_paged.cu — attention over a paged key-value cache: one new token per sequence, or the tokens of a
// prompt chunk with a sliding window and first rows that stay visible.
//
// Mathematics: o_h = sum_j exp(s_hj - lse_h) k_j with s_hj = scale q_h . k_j over the visible rows j and
// lse_h = log(sum_j exp(s_hj) + exp(sink_h)).  One row is key and value of every head (the reference's
// cache has one KV head; cuda/flash_attn.cu:148-313).
#include "device_utils.cuh"
#include "kernels.cuh"

namespace ds4b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The rows one token sees, as a list: the first `n_first`, then lo .. p.
struct Seen {
    int first, lo, n;
    __device__ __forceinline__ int row(int i) const { return i < first ? i : lo + (i - first); }
};
__device__ __forceinline__ Seen seen_rows(int p, int window, int n_first) {
    Seen s;
    s.lo = window > 0 && p + 1 > window ? p + 1 - window : 0;
    s.first = min(n_first, s.lo);
    s.n = p < 0 ? 0 : s.first + (p + 1 - s.lo);
    return s;
}

// ---------------------------------------------------------------------------- one warp per head, f32
constexpr int kSimpleWarps = 8;

template <int V>      // float4s of a row per lane: head_dim / 128
__global__ void __launch_bounds__(kSimpleWarps * 32) attn_rows_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 31, h = (int)blockIdx.y * kSimpleWarps + (threadIdx.x >> 5);
    const int64_t t = blockIdx.x;
    if (h >= a.n_heads) return;
    const int dim = a.kv.head_dim;
    const int64_t most = a.table_width * a.kv.page_rows;
    int b, p;
    if (a.q_start) {
        if (t < a.q_start[0] || t >= a.q_start[a.n_seqs]) return;
        int lo = 0, hi = a.n_seqs - 1;              // the last sequence that starts at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.q_start[mid] <= t) lo = mid; else hi = mid - 1;
        }
        b = lo;
        p = (int)min((int64_t)a.kv_len[b], most) - a.q_start[b + 1] + (int)t;
    } else {
        b = (int)t;
        p = (int)min((int64_t)a.kv_len[b], most) - 1;
    }
    const Seen seen = seen_rows(p, a.window, a.n_first);
    const uint16_t *qr = a.q + (t * a.n_heads + h) * dim;
    float4 q[V], o[V];
    const float k = a.scale * kLog2e;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint2 u = __ldg(reinterpret_cast<const uint2 *>(qr + 4 * (lane + 32 * j)));
        q[j] = make_float4(__uint_as_float(u.x << 16) * k, __uint_as_float(u.x & 0xffff0000u) * k,
                           __uint_as_float(u.y << 16) * k, __uint_as_float(u.y & 0xffff0000u) * k);
        o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY, l = 0.0f;
    for (int i = 0; i < seen.n; ++i) {
        const int row = seen.row(i);
        const int page = a.page_table[b * a.table_width + row / a.kv.page_rows];
        if (page < 0 || page >= a.kv.n_pages) continue;
        const int64_t slot = (int64_t)page * a.kv.page_rows + row % a.kv.page_rows;
        float4 r[V];
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int e = 4 * (lane + 32 * j);
            if (a.kv.row_format == DS4B200_KV_F32) {
                r[j] = ld_ro4(a.kv.raw + slot * dim + e);
            } else {
                const int nope = dim - a.kv.n_rot;
                if (a.kv.row_format == DS4B200_KV_FP8_BLOCK64 && e >= nope) {
                    r[j] = ld_ro4(a.kv.tail + slot * a.kv.n_rot + (e - nope));
                } else {
                    const uint32_t c = __ldg(reinterpret_cast<const uint32_t *>(a.kv.codes + slot * dim + e));
                    const float sc = a.kv.row_format == DS4B200_KV_FP8_ROW ? __ldg(a.kv.scales + slot)
                                                                           : __ldg(a.kv.scales + slot * (nope >> 6) + (e >> 6));
                    const float2 x = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xffff), __NV_E4M3)));
                    const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3)));
                    r[j] = make_float4(x.x * sc, x.y * sc, y.x * sc, y.y * sc);
                }
            }
            s += q[j].x * r[j].x + q[j].y * r[j].y + q[j].z * r[j].z + q[j].w * r[j].w;
        }
        s = warp_sum(s);
        const float m2 = fmaxf(m, s), c = exp2f(m - m2), w = exp2f(s - m2);
        l = l * c + w;
        m = m2;
#pragma unroll
        for (int j = 0; j < V; ++j)
            o[j] = make_float4(o[j].x * c + w * r[j].x, o[j].y * c + w * r[j].y, o[j].z * c + w * r[j].z, o[j].w * c + w * r[j].w);
    }
    if (a.sink) {
        const float s = a.sink[h] * kLog2e, m2 = fmaxf(m, s);
        const float c = m == -INFINITY ? 0.0f : exp2f(m - m2);
        l = l * c + (s == -INFINITY ? 0.0f : exp2f(s - m2));
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = make_float4(o[j].x * c, o[j].y * c, o[j].z * c, o[j].w * c);
        m = m2;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (lane == 0 && a.lse) a.lse[t * a.n_heads + h] = l > 0.0f ? (m + log2f(l)) / kLog2e : -INFINITY;
    uint16_t *orow = a.out + (t * a.n_heads + h) * dim;
#pragma unroll
    for (int j = 0; j < V; ++j)
        st_bf16x4(orow + 4 * (lane + 32 * j), make_float4(o[j].x * inv, o[j].y * inv, o[j].z * inv, o[j].w * inv));
}

}  // namespace

int64_t attn_workspace_bytes(int n_heads, int head_dim) { return 16; }

void attn_paged(const AttnArgs &a, cudaStream_t s) {
    const dim3 grid((unsigned)a.n_tokens, (unsigned)((a.n_heads + kSimpleWarps - 1) / kSimpleWarps));
    switch (a.kv.head_dim / 128) {
        case 1: attn_rows_kernel<1><<<grid, kSimpleWarps * 32, 0, s>>>(a); break;
        case 2: attn_rows_kernel<2><<<grid, kSimpleWarps * 32, 0, s>>>(a); break;
        case 3: attn_rows_kernel<3><<<grid, kSimpleWarps * 32, 0, s>>>(a); break;
        default: attn_rows_kernel<4><<<grid, kSimpleWarps * 32, 0, s>>>(a); break;
    }
}

}  // namespace ds4b200
