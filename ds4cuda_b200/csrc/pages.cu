// pages.cu — copying, forking, reserving, freeing and compacting the pages of a cache pool.
//
// Every call is one planning kernel of a single CTA and one kernel over the whole card.  The plan checks the
// list, scans the reference counts for free pages (ascending, so the pages handed out do not depend on timing)
// and leaves a list of page moves in the workspace; the second kernel rewrites the tables and moves the
// pages.  A pool's counts are a few KiB to a few hundred KiB, so one CTA reads them in microseconds, and a
// plan spread over CTAs would need a grid-wide scan with its own round trips.
//
// The move kernel is bound by HBM (2 bytes of traffic per byte moved): units of 16 KiB, four 128-bit loads in
// flight per thread, eight CTAs per SM.
#include "device_utils.cuh"
#include "kernels.cuh"

namespace ds4b200 {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kUnitBytes = kMoveThreads * 16 * 4;     // 16 KiB
constexpr int kMoveCtas = 148 * 8;

struct Header { int status, n_moves, pad[2]; };

// the workspace, in this order
struct Work {
    Header *head;
    int *mark;       // per sequence: fork 1 + its pair's index, free 1 + its pages (0 = not listed), reserve its pages before
    int *first;      // per list entry or sequence: rank of its first new page
    int *fresh;      // new pages in ascending order
    int2 *moves;
    int *map;        // per page: where it goes (compact), or how often it is written (copy)
};

struct Tables {
    const int *refs_in; int *refs_out;
    const int *table_in; int *table_out;
    const int *lens_in; int *lens_out;
    int64_t n_pages, n_seqs, width;
    int page_rows;
};

struct ArrayList {
    int n;
    int units_total;                               // units of one page over all arrays
    bool wide;                                     // every base and page size a multiple of 16
    unsigned char *base[kMaxPageArrays];
    int64_t page_bytes[kMaxPageArrays];
    int unit_first[kMaxPageArrays + 1];
};

__device__ __forceinline__ int64_t pages_of(int64_t rows, int page_rows) { return (rows + page_rows - 1) / page_rows; }

// Exclusive prefix sum over the CTA's threads; *total gets the sum.  scratch: 33 ints.
__device__ __forceinline__ int block_scan(int v, int *scratch, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int t = lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0;
        const int own = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, t, o); if (lane >= o) t += y; }
        scratch[lane] = t - own;
        if (lane == 31) scratch[32] = t;
    }
    __syncthreads();
    const int r = scratch[warp] + x - v;
    *total = scratch[32];
    __syncthreads();
    return r;
}

// refs_out = refs_in, and the `need` free pages of lowest index to fresh[] (as many as there are);
// returns how many free pages were seen, capped at `need`.
__device__ int collect_free(const Tables &t, int need, int *fresh, int *scratch) {
    int found = 0;
    for (int64_t base = 0; base < t.n_pages && found < need; base += kPlanThreads) {
        const int64_t p = base + threadIdx.x;
        const int is_free = p < t.n_pages && t.refs_in[p] <= 0;
        int total;
        const int r = found + block_scan(is_free, scratch, &total);
        if (is_free && r < need) fresh[r] = (int)p;
        found += total;
    }
    return found < need ? found : need;
}
__device__ __forceinline__ void copy_refs(const Tables &t) {
    if (t.refs_out != t.refs_in)
        for (int64_t p = threadIdx.x; p < t.n_pages; p += kPlanThreads) t.refs_out[p] = t.refs_in[p];
}

__global__ void __launch_bounds__(kPlanThreads) plan_fork_kernel(Tables t, const int2 *pairs, int n_pairs, Work w, int *status) {
    __shared__ int scratch[33];
    __shared__ int bad;
    launch_dependents();
    const int tid = threadIdx.x;
    if (tid == 0) bad = 0;
    for (int64_t s = tid; s < t.n_seqs; s += kPlanThreads) w.mark[s] = 0;
    __syncthreads();
    for (int i = tid; i < n_pairs; i += kPlanThreads) {
        const int2 pr = pairs[i];
        const bool in = pr.x >= 0 && pr.x < t.n_seqs && pr.y >= 0 && pr.y < t.n_seqs;
        if (!in || atomicCAS(&w.mark[in ? pr.y : 0], 0, i + 1) != 0) bad = 1;
    }
    __syncthreads();
    if (!bad) {                                     // a target is nobody's source; the source's pages exist
        for (int i = tid >> 5; i < n_pairs; i += kPlanThreads >> 5) {
            const int src = pairs[i].x;
            const int len = t.lens_in[src];
            bool ok = w.mark[src] == 0 && len >= 0 && len <= t.width * t.page_rows;
            if (ok) {
                const int n = (int)pages_of(len, t.page_rows);
                for (int c = tid & 31; c < n; c += 32) {
                    const int p = t.table_in[src * t.width + c];
                    ok = ok && p >= 0 && p < t.n_pages;
                }
            }
            if (!ok) bad = 1;
        }
    }
    __syncthreads();
    int need = 0;
    if (!bad)
        for (int base = 0; base < n_pairs; base += kPlanThreads) {
            const int i = base + tid;
            const int part = i < n_pairs && t.lens_in[pairs[i].x] % t.page_rows != 0;
            int total;
            const int r = need + block_scan(part, scratch, &total);
            if (i < n_pairs) w.first[i] = part ? r : -1;
            need += total;
        }
    const int found = bad ? 0 : collect_free(t, need, w.fresh, scratch);
    __syncthreads();
    const int st = bad ? -1 : need - found;
    copy_refs(t);
    __syncthreads();
    if (st == 0)
        for (int i = tid; i < n_pairs; i += kPlanThreads) {
            const int r = w.first[i];
            if (r < 0) continue;
            const int src = pairs[i].x, page = w.fresh[r];
            w.moves[r] = make_int2(t.table_in[src * t.width + t.lens_in[src] / t.page_rows], page);
            t.refs_out[page] = 1;
        }
    for (int64_t s = tid; s < t.n_seqs; s += kPlanThreads)   // a source's length is no target's: in place is fine
        t.lens_out[s] = st == 0 && w.mark[s] ? t.lens_in[pairs[w.mark[s] - 1].x] : t.lens_in[s];
    if (tid == 0) { w.head->status = st; w.head->n_moves = st == 0 ? need : 0; *status = st; }
}

__global__ void __launch_bounds__(kPlanThreads) plan_reserve_kernel(Tables t, const int *new_lens, Work w, int *status) {
    __shared__ int scratch[33];
    __shared__ int bad;
    __shared__ unsigned long long asked;
    launch_dependents();
    const int tid = threadIdx.x;
    if (tid == 0) { bad = 0; asked = 0; }
    __syncthreads();
    int64_t need = 0, mine = 0;                     // pages: of the sequences before these, cut at the pool's size; of this thread's, all
    const int64_t most = t.width * t.page_rows;
    for (int64_t base = 0; base < t.n_seqs; base += kPlanThreads) {
        const int64_t b = base + tid;
        int k = 0;
        if (b < t.n_seqs) {
            const int64_t len = t.lens_in[b], want = max(len, (int64_t)new_lens[b]);
            if (len < 0 || want > most) bad = 1;
            else {
                const int64_t more = pages_of(want, t.page_rows) - pages_of(len, t.page_rows);
                k = (int)min(more, t.n_pages + 1);
                mine += more;
            }
            if (!bad) w.mark[b] = (int)pages_of(len, t.page_rows);
        }
        int total;
        const int r = block_scan(k, scratch, &total);
        // a sum past the pool's size only has to stay past it (n_pages <= 2^20: 1024 of them fit an int)
        if (b < t.n_seqs) w.first[b] = (int)min(need + r, t.n_pages);
        need += total;
    }
    atomicAdd(&asked, (unsigned long long)mine);
    __syncthreads();
    const int ask = (int)min(need, t.n_pages);
    const int found = bad ? 0 : collect_free(t, ask, w.fresh, scratch);
    __syncthreads();
    const int st = bad ? -1 : (int)min((int64_t)asked - found, (int64_t)0x7fffffff);
    copy_refs(t);
    __syncthreads();
    if (st == 0)
        for (int i = tid; i < ask; i += kPlanThreads) t.refs_out[w.fresh[i]] = 1;
    for (int64_t b = tid; b < t.n_seqs; b += kPlanThreads) {
        const int len = t.lens_in[b];
        t.lens_out[b] = st == 0 ? max(len, new_lens[b]) : len;
    }
    if (tid == 0) { w.head->status = st; w.head->n_moves = 0; *status = st; }
}

__global__ void __launch_bounds__(kPlanThreads) plan_free_kernel(Tables t, const int *seqs, int n_list, Work w, int *status) {
    __shared__ int bad;
    launch_dependents();
    const int tid = threadIdx.x;
    if (tid == 0) bad = 0;
    for (int64_t s = tid; s < t.n_seqs; s += kPlanThreads) w.mark[s] = 0;
    __syncthreads();
    for (int i = tid; i < n_list; i += kPlanThreads) {
        const int s = seqs[i];
        if (s < 0 || s >= t.n_seqs) bad = 1;
        else w.mark[s] = 1;
    }
    __syncthreads();
    if (!bad)
        for (int i = tid >> 5; i < n_list; i += kPlanThreads >> 5) {
            const int s = seqs[i], len = t.lens_in[s];
            bool ok = len >= 0 && len <= t.width * t.page_rows;
            if (ok) {
                const int n = (int)pages_of(len, t.page_rows);
                for (int c = tid & 31; c < n; c += 32) {
                    const int p = t.table_in[s * t.width + c];
                    ok = ok && p >= 0 && p < t.n_pages;
                }
            }
            if (!ok) bad = 1;
        }
    __syncthreads();
    copy_refs(t);
    for (int64_t s = tid; s < t.n_seqs; s += kPlanThreads) {
        const int len = t.lens_in[s];
        const bool gone = !bad && w.mark[s];
        if (gone) w.mark[s] = 1 + (int)pages_of(len, t.page_rows);
        t.lens_out[s] = gone ? 0 : len;
    }
    if (tid == 0) { w.head->status = bad ? -1 : 0; w.head->n_moves = 0; *status = bad ? -1 : 0; }
}

__global__ void __launch_bounds__(kPlanThreads) plan_compact_kernel(Tables t, Work w, int *n_live) {
    __shared__ int scratch[33];
    launch_dependents();
    const int tid = threadIdx.x;
    int live = 0;
    for (int64_t p = tid; p < t.n_pages; p += kPlanThreads) live += t.refs_in[p] > 0;
    int n;
    block_scan(live, scratch, &n);
    int holes = 0, high = 0;
    for (int64_t base = 0; base < t.n_pages; base += kPlanThreads) {
        const int64_t p = base + tid;
        const int ref = p < t.n_pages ? t.refs_in[p] : 0;
        const int is_hole = p < n && ref <= 0, is_high = p >= n && p < t.n_pages && ref > 0;
        // one scan for both: at most 1024 of each in a round, so they share a word
        int total;
        const int r = block_scan(is_hole | (is_high << 16), scratch, &total);
        if (is_hole) w.moves[holes + (r & 0xffff)].y = (int)p;
        if (is_high) w.moves[high + (r >> 16)].x = (int)p;
        if (p < t.n_pages) {
            w.map[p] = (int)p;
            t.refs_out[p] = ref > 0 ? ref : 0;
        }
        holes += total & 0xffff;
        high += total >> 16;
    }
    __syncthreads();
    for (int i = tid; i < high; i += kPlanThreads) {        // holes == high
        const int2 m = w.moves[i];
        w.map[m.x] = m.y;
        t.refs_out[m.y] = t.refs_out[m.x];
        t.refs_out[m.x] = 0;
    }
    if (tid == 0) { w.head->status = 0; w.head->n_moves = high; *n_live = n; }
}

__global__ void __launch_bounds__(kPlanThreads) plan_copy_kernel(const int2 *moves, int n_moves, int64_t n_pages, Work w, int *status) {
    __shared__ int bad;
    launch_dependents();
    const int tid = threadIdx.x;
    if (tid == 0) bad = 0;
    for (int64_t p = tid; p < n_pages; p += kPlanThreads) w.map[p] = 0;
    __syncthreads();
    for (int i = tid; i < n_moves; i += kPlanThreads) {
        const int2 m = moves[i];
        const bool in = m.x >= 0 && m.x < n_pages && m.y >= 0 && m.y < n_pages;
        if (!in || atomicCAS(&w.map[in ? m.y : 0], 0, 1) != 0) bad = 1;
    }
    __syncthreads();
    if (!bad)
        for (int i = tid; i < n_moves; i += kPlanThreads) {
            if (w.map[moves[i].x] != 0) bad = 1;            // a written page is nobody's source
            w.moves[i] = moves[i];
        }
    __syncthreads();
    if (tid == 0) { w.head->status = bad ? -1 : 0; w.head->n_moves = bad ? 0 : n_moves; *status = bad ? -1 : 0; }
}

enum { kFork, kReserve, kFree, kCompact, kCopy };

template <bool WIDE>
__device__ __forceinline__ void move_unit(const unsigned char *src, unsigned char *dst, int64_t bytes) {
    using V = typename std::conditional<WIDE, uint4, uint32_t>::type;
    const int n = (int)(bytes / sizeof(V));
    const V *s = reinterpret_cast<const V *>(src);
    V *d = reinterpret_cast<V *>(dst);
    for (int base = 0; base < n; base += 4 * kMoveThreads) {
        V v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + j * kMoveThreads + (int)threadIdx.x;
            if (i < n) v[j] = __ldcs(s + i);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = base + j * kMoveThreads + (int)threadIdx.x;
            if (i < n) __stcs(d + i, v[j]);
        }
    }
}

template <int OP>
__global__ void __launch_bounds__(kMoveThreads) apply_kernel(Tables t, const int2 *pairs, Work w,
                                                             const __grid_constant__ ArrayList a) {
    wait_dependency();
    const bool done = w.head->status == 0;
    const int64_t step = (int64_t)gridDim.x * kMoveThreads, me = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x;
    if (OP != kCopy) {
        for (int64_t i = me; i < t.n_seqs * t.width; i += step) {
            const int64_t s = i / t.width;
            const int c = (int)(i - s * t.width);
            int v = t.table_in[i];
            if (OP == kFork && done && w.mark[s]) {
                const int k = w.mark[s] - 1, src = pairs[k].x, full = t.lens_in[src] / t.page_rows;
                v = -1;
                if (c < full) {
                    v = t.table_in[src * t.width + c];
                    atomicAdd(&t.refs_out[v], 1);
                } else if (c == full && w.first[k] >= 0) {
                    v = w.fresh[w.first[k]];
                }
            }
            if (OP == kReserve && done) {
                const int have = w.mark[s];                 // pages before the call
                if (c >= have && c < pages_of(t.lens_out[s], t.page_rows)) v = w.fresh[w.first[s] + (c - have)];
            }
            if (OP == kFree && done && w.mark[s]) {
                if (c < w.mark[s] - 1) atomicSub(&t.refs_out[v], 1);
                v = -1;
            }
            if (OP == kCompact && v >= 0 && v < t.n_pages) v = w.map[v];
            t.table_out[i] = v;
        }
    }
    if (OP == kFork || OP == kCompact || OP == kCopy) {
        const int64_t units = (int64_t)w.head->n_moves * a.units_total;
        for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
            const int m = (int)(u / a.units_total), r = (int)(u - (int64_t)m * a.units_total);
            int lo = 0, hi = a.n - 1;                       // the array this unit lies in
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (a.unit_first[mid] <= r) lo = mid; else hi = mid - 1;
            }
            const int2 mv = w.moves[m];
            const int64_t off = (int64_t)(r - a.unit_first[lo]) * kUnitBytes;
            const int64_t bytes = min((int64_t)kUnitBytes, a.page_bytes[lo] - off);
            const unsigned char *src = a.base[lo] + (int64_t)mv.x * a.page_bytes[lo] + off;
            unsigned char *dst = a.base[lo] + (int64_t)mv.y * a.page_bytes[lo] + off;
            if (a.wide) move_unit<true>(src, dst, bytes);
            else move_unit<false>(src, dst, bytes);
        }
    }
}

constexpr int64_t round16(int64_t b) { return (b + 15) / 16 * 16; }

Work lay_out(void *ws, int64_t n_pages, int64_t n_seqs, int64_t n_list) {
    Work w;
    unsigned char *p = static_cast<unsigned char *>(ws);
    const int64_t n = n_list > n_seqs ? n_list : n_seqs;
    w.head = reinterpret_cast<Header *>(p); p += sizeof(Header);
    w.mark = reinterpret_cast<int *>(p); p += round16(4 * n_seqs);
    w.first = reinterpret_cast<int *>(p); p += round16(4 * n);
    w.fresh = reinterpret_cast<int *>(p); p += round16(4 * n_pages);
    w.map = reinterpret_cast<int *>(p); p += round16(4 * n_pages);
    w.moves = reinterpret_cast<int2 *>(p);
    return w;
}

ArrayList list_arrays(const ds4b200_page_array *host, int n) {
    ArrayList a;
    a.n = n;
    a.wide = true;
    int units = 0;
    for (int i = 0; i < n; ++i) {
        a.base[i] = static_cast<unsigned char *>(host[i].base);
        a.page_bytes[i] = host[i].page_bytes;
        a.unit_first[i] = units;
        units += (int)((host[i].page_bytes + kUnitBytes - 1) / kUnitBytes);
        a.wide = a.wide && aligned16(host[i].base) && host[i].page_bytes % 16 == 0;
    }
    a.unit_first[n] = units;
    a.units_total = units;
    return a;
}

unsigned small_grid(int64_t n) {
    const int64_t g = (n + kMoveThreads - 1) / kMoveThreads;
    return (unsigned)(g < 1 ? 1 : g < kMoveCtas ? g : kMoveCtas);
}

}  // namespace

int64_t pages_workspace_bytes(int64_t n_pages, int64_t n_seqs, int64_t n_list) {
    const int64_t n = n_list > n_seqs ? n_list : n_seqs, m = n_list > n_pages ? n_list : n_pages;
    return (int64_t)sizeof(Header) + round16(4 * n_seqs) + round16(4 * n) + 2 * round16(4 * n_pages) + 8 * m;
}

void pages_copy(const ds4b200_page_array *host, int n_arrays, int64_t n_pages, const int32_t *moves, int64_t n_moves,
                int32_t *status, void *ws, cudaStream_t s) {
    const Work w = lay_out(ws, n_pages, 0, n_moves);
    const ArrayList a = list_arrays(host, n_arrays);
    const int2 *mv = reinterpret_cast<const int2 *>(moves);
    plan_copy_kernel<<<1, kPlanThreads, 0, s>>>(mv, (int)n_moves, n_pages, w, status);
    launch_behind(apply_kernel<kCopy>, kMoveCtas, kMoveThreads, 0, s, Tables{}, mv, w, a);
}

void pages_fork(const ds4b200_page_array *host, int n_arrays, const PageTables &p, const int32_t *pairs, int64_t n_pairs,
                int32_t *status, void *ws, cudaStream_t s) {
    const Tables t{p.refs_in, p.refs_out, p.table_in, p.table_out, p.lens_in, p.lens_out, p.n_pages, p.n_seqs, p.width, p.page_rows};
    const Work w = lay_out(ws, p.n_pages, p.n_seqs, n_pairs);
    const ArrayList a = list_arrays(host, n_arrays);
    const int2 *pr = reinterpret_cast<const int2 *>(pairs);
    plan_fork_kernel<<<1, kPlanThreads, 0, s>>>(t, pr, (int)n_pairs, w, status);
    launch_behind(apply_kernel<kFork>, kMoveCtas, kMoveThreads, 0, s, t, pr, w, a);
}

void pages_reserve(const PageTables &p, const int32_t *new_lens, int32_t *status, void *ws, cudaStream_t s) {
    const Tables t{p.refs_in, p.refs_out, p.table_in, p.table_out, p.lens_in, p.lens_out, p.n_pages, p.n_seqs, p.width, p.page_rows};
    const Work w = lay_out(ws, p.n_pages, p.n_seqs, 0);
    plan_reserve_kernel<<<1, kPlanThreads, 0, s>>>(t, new_lens, w, status);
    launch_behind(apply_kernel<kReserve>, small_grid(p.n_seqs * p.width), kMoveThreads, 0, s, t, (const int2 *)nullptr, w, ArrayList{});
}

void pages_free(const PageTables &p, const int32_t *seqs, int64_t n_list, int32_t *status, void *ws, cudaStream_t s) {
    const Tables t{p.refs_in, p.refs_out, p.table_in, p.table_out, p.lens_in, p.lens_out, p.n_pages, p.n_seqs, p.width, p.page_rows};
    const Work w = lay_out(ws, p.n_pages, p.n_seqs, n_list);
    plan_free_kernel<<<1, kPlanThreads, 0, s>>>(t, seqs, (int)n_list, w, status);
    launch_behind(apply_kernel<kFree>, small_grid(p.n_seqs * p.width), kMoveThreads, 0, s, t, (const int2 *)nullptr, w, ArrayList{});
}

void pages_compact(const ds4b200_page_array *host, int n_arrays, const PageTables &p, int32_t *n_live, void *ws, cudaStream_t s) {
    const Tables t{p.refs_in, p.refs_out, p.table_in, p.table_out, nullptr, nullptr, p.n_pages, p.n_seqs, p.width, 1};
    const Work w = lay_out(ws, p.n_pages, p.n_seqs, 0);
    const ArrayList a = list_arrays(host, n_arrays);
    plan_compact_kernel<<<1, kPlanThreads, 0, s>>>(t, w, n_live);
    launch_behind(apply_kernel<kCompact>, kMoveCtas, kMoveThreads, 0, s, t, (const int2 *)nullptr, w, a);
}

}  // namespace ds4b200
