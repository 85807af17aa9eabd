// The pages of a paged cache: room for new tokens (extend), branches that share their prefix (fork), pages given back
// (free, trim) and pages in use moved to the front (compact).
//
// State on the device: page_table [rows, max_pages] (physical page of each logical page, -1 = none), seq_lens [rows],
// refs [num_pages] = table entries that name a page.  A page is free when refs is 0; new pages are always the lowest free
// ones, in the order of the calls' rows, so that results do not depend on scheduling.  No call reads anything back to the
// host: all of them can be captured.
//
// Allocation and compaction need ranks over `refs` (the k-th free page): every warp counts a contiguous slice, the counts are
// exchanged, and the slices are walked again with the ranks known.  Up to kOneCta pages one CTA does it (its barriers cost 30
// ns), beyond a cluster of eight (1.2 us per exchange, eight times the loads in flight).  What follows -- table rows, page
// data -- is a second launch over all SMs, chained programmatically.  Bound by latency at small sizes, by memory (page data,
// read once and written once) at large ones.
#include "msk.h"
#include "ptx.cuh"

namespace msk {
namespace {

constexpr int kCluster = 8;
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kOneCta = 16384;        // pages (free + extend of 16 rows, one CTA / cluster: 4096 pages 9.2 / 13.0 us, 65536 18.6 / 13.8)
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = 16384;     // bytes a CTA moves at a time: 4 x 16 per thread in flight
constexpr int kMaxCaches = 128;
constexpr int kWhere = MSK_K_PAGES << 8;

struct Caches {
    uint8_t* p[kMaxCaches];
    int n;
    int token_bytes;
};

struct PlanArgs {
    int* page_table;
    int* seq_lens;
    int* refs;
    int rows, max_pages, num_pages, page_size, page_log;
    const int* list;       // rows to extend / children
    const int* parents;    // fork
    int n;
    int q_len;             // extend: tokens per row, or
    const int* cu;         // ... cu[n + 1]
    int tokens;            // entries of cache_loc
    long long* cache_loc;
    // workspace
    int* counts;           // [3][kCluster * kPlanWarps] slices' counts, then [4]: results
    int* claim;            // [rows] first list entry that names a row
    int* is_parent;        // [rows]
    int* need;             // [n]
    int* offs;             // [n]
    int* free_list;        // [num_pages]
    int4* ops;             // [n] fork: source page, new page, tokens to copy, 1 = done / 0 = refused / 2 = no page
    int* src;              // [num_pages] compact: moved pages ...
    int* dst;              // ... and where to
    int* remap;            // [num_pages]
    int* result;           // compact: pages in use, pages moved; or NULL
    int* status;
};

// (exclusive prefix of v over the CTA's threads, total) -- kPlanThreads threads.
__device__ __forceinline__ int block_scan(int v, int* total) {
    __shared__ int part[kPlanWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();  // the previous call's readers are done
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    const int w = part[lane];
    int winc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc += u;
    }
    *total = __shfl_sync(0xffffffffu, winc, 31);
    const int before = __shfl_sync(0xffffffffu, winc - w, warp);
    return before + inc - v;
}

// Everything written so far, global memory included, is visible to all planning threads after it.
__device__ __forceinline__ void exchange(int nct) {
    if (nct == 1) {
        __syncthreads();
    } else {
        __threadfence();
        cluster_sync_all();
    }
}

// Walks the pages [lo, hi) of `refs` with one warp, four per lane and step: f(first page, r[4], how many).
template <class F>
__device__ __forceinline__ void walk_refs(const int* refs, int lo, int hi, F f) {
    const int lane = threadIdx.x & 31;
#pragma unroll 4
    for (int at = lo; at < hi; at += 128) {
        const int i = at + 4 * lane;
        int r[4] = {0, 0, 0, 0};
        const int k = min(max(hi - i, 0), 4);
        if (k == 4 && (reinterpret_cast<uintptr_t>(refs + i) & 15) == 0) {
            const int4 v = __ldcg(reinterpret_cast<const int4*>(refs + i));
            r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
        } else {
            for (int j = 0; j < k; ++j) r[j] = __ldcg(refs + i + j);
        }
        f(i, r, k);
    }
}

__device__ __forceinline__ void slice_of(const PlanArgs& p, int gwarp, int nwarps, int* lo, int* hi) {  // multiples of a step
    const int per = ((p.num_pages + nwarps - 1) / nwarps + 127) & ~127;
    *lo = static_cast<int>(min(static_cast<long long>(gwarp) * per, static_cast<long long>(p.num_pages)));
    *hi = static_cast<int>(min(static_cast<long long>(*lo) + per, static_cast<long long>(p.num_pages)));
}

__device__ __forceinline__ int warp_total(int v) { return __reduce_add_sync(0xffffffffu, v); }
__device__ __forceinline__ int lanes_before(int v) {  // sum over the lower lanes
    const int lane = threadIdx.x & 31;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    return inc - v;
}
// (sum of the counts of all slices, of those before slice gwarp) -- a whole warp.
__device__ __forceinline__ int slice_total(const int* counts, int gwarp, int nwarps, int* before) {
    const int lane = threadIdx.x & 31;
    int all = 0, low = 0;
    for (int w = lane; w < nwarps; w += 32) {
        const int v = __ldcg(counts + w);
        all += v;
        if (w < gwarp) low += v;
    }
    *before = warp_total(low);
    return warp_total(all);
}

// The new tokens of list entry j: how many, and where they begin in cache_loc; false where cu_seqlens falls or names more
// tokens than there are (then those that cache_loc has).
__device__ __forceinline__ bool tokens_of(const PlanArgs& p, int j, int* n_tok, int* first_loc) {
    if (p.cu == nullptr) {
        *first_loc = j * p.q_len, *n_tok = p.q_len;
        return true;
    }
    const int a = p.cu[j], b = p.cu[j + 1];
    *first_loc = min(max(a, 0), p.tokens), *n_tok = max(min(max(b, 0), p.tokens) - *first_loc, 0);
    return 0 <= a && a <= b && b <= p.tokens;
}

// A page that new tokens of a row must not go into: another row holds it too, or there is no such page.
__device__ __forceinline__ bool not_its_own(const PlanArgs& p, int id) { return id >= p.num_pages || (id >= 0 && __ldcg(p.refs + id) > 1); }

// One CTA or one cluster: gives list entries the free pages they need.  kFork: one page for a child whose parent ends inside a page.
template <bool kFork>
__global__ void __launch_bounds__(kPlanThreads) pages_plan_kernel(PlanArgs p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, nct = gridDim.x;  // one CTA, or the one cluster
    const int gtid = rank * kPlanThreads + tid, gwarp = rank * kPlanWarps + warp;
    const int kAll = nct * kPlanThreads, kAllWarps = nct * kPlanWarps;
    pdl_wait();
    pdl_launch_dependents();
    // which list entry speaks for a row: the first that names it
    for (int r = gtid; r < p.rows; r += kAll) {
        p.claim[r] = 0x7fffffff;
        if (kFork) p.is_parent[r] = 0;
    }
    int lo, hi;
    slice_of(p, gwarp, kAllWarps, &lo, &hi);
    int mine = 0;
    walk_refs(p.refs, lo, hi, [&](int, const int (&r)[4], int k) {
        for (int j = 0; j < 4; ++j) mine += j < k && r[j] == 0;
    });
    mine = warp_total(mine);
    if (lane == 0) p.counts[gwarp] = mine;
    exchange(nct);
    for (int j = gtid; j < p.n; j += kAll) {
        const int row = p.list[j];
        if (row >= 0 && row < p.rows) atomicMin(p.claim + row, j);
        if (kFork) {
            const int par = p.parents[j];
            if (par >= 0 && par < p.rows) atomicExch(p.is_parent + par, 1);
        }
    }
    exchange(nct);
    // what each entry needs: a thread per entry where it is few pages, else a warp per entry and a lane per page
    const bool few = kFork || (p.cu == nullptr && p.q_len <= 4 * p.page_size);
    if (few) {
        for (int j = gtid; j < p.n; j += kAll) {
            const int row = p.list[j];
            bool ok = row >= 0 && row < p.rows && __ldcg(p.claim + row) == j;
            int need = 0;
            if (kFork) {
                const int par = p.parents[j];
                ok = ok && par >= 0 && par < p.rows && __ldcg(p.is_parent + row) == 0;
                int4 op = make_int4(-1, -1, 0, 0);
                if (ok) {
                    const int seq = p.seq_lens[par], full = seq >> p.page_log, part = seq & (p.page_size - 1);
                    if (seq >= 0 && full + (part > 0) <= p.max_pages) {
                        op.w = 1;
                        if (part > 0) {
                            op.x = p.page_table[static_cast<size_t>(par) * p.max_pages + full];
                            op.z = part;
                            if (op.x >= p.num_pages) report(p.status, MSK_ERR_BOUNDS, kWhere | 6, op.x, p.num_pages);
                            if (op.x >= p.num_pages || op.x < 0) op.x = -1;
                            need = op.x >= 0;
                        }
                    }
                }
                if (op.w == 0) report(p.status, MSK_ERR_BOUNDS, kWhere | 1, row, j);
                p.ops[j] = op;
            } else if (ok) {
                const int seq = p.seq_lens[row];
                ok = seq >= 0;
                if (!ok) report(p.status, MSK_ERR_BOUNDS, kWhere | 9, seq, row);
                const int last = static_cast<int>((static_cast<long long>(seq) + p.q_len - 1) >> p.page_log);
                if (ok && p.q_len > 0 && last >= p.max_pages) report(p.status, MSK_ERR_CAPACITY, kWhere | 3, last, p.max_pages);
                if (ok && p.q_len > 0)
                    for (int lp = seq >> p.page_log; lp <= min(last, p.max_pages - 1); ++lp) {
                        const int id = p.page_table[static_cast<size_t>(row) * p.max_pages + lp];
                        need += id < 0;
                        if (not_its_own(p, id)) {
                            report(p.status, MSK_ERR_BOUNDS, kWhere | 7, id, row);
                            ok = false;
                        }
                    }
            } else {
                report(p.status, MSK_ERR_BOUNDS, kWhere | 2, row, j);
            }
            p.need[j] = ok ? need : (kFork ? 0 : -1);  // extend: -1 = refused
        }
    } else {
        for (int j = gwarp; j < p.n; j += kAllWarps) {
            const int row = p.list[j];
            bool ok = row >= 0 && row < p.rows && __ldcg(p.claim + row) == j;
            int need = 0;
            if (!ok && lane == 0) report(p.status, MSK_ERR_BOUNDS, kWhere | 2, row, j);
            int n_tok, first_loc;
            if (!tokens_of(p, j, &n_tok, &first_loc)) {
                if (lane == 0) report(p.status, MSK_ERR_BOUNDS, kWhere | 8, p.cu[j + 1], p.tokens);
                ok = false;
            }
            if (ok) {
                const int seq = p.seq_lens[row];
                ok = seq >= 0;
                if (!ok && lane == 0) report(p.status, MSK_ERR_BOUNDS, kWhere | 9, seq, row);
                const int first = seq >> p.page_log;
                const int last = n_tok > 0 ? static_cast<int>((static_cast<long long>(seq) + n_tok - 1) >> p.page_log) : first - 1;
                if (ok && last >= p.max_pages && lane == 0) report(p.status, MSK_ERR_CAPACITY, kWhere | 3, last, p.max_pages);
                const int end = ok ? min(last, p.max_pages - 1) : first - 1;
                for (int lp0 = first; lp0 <= end; lp0 += 32) {
                    const int lp = lp0 + lane;
                    const int id = lp <= end ? p.page_table[static_cast<size_t>(row) * p.max_pages + lp] : 0x80000000;
                    need += __popc(__ballot_sync(0xffffffffu, lp <= end && id < 0));
                    const uint32_t bad = __ballot_sync(0xffffffffu, not_its_own(p, id));
                    if (bad != 0 && lane == __ffs(bad) - 1) report(p.status, MSK_ERR_BOUNDS, kWhere | 7, id, row);
                    ok = ok && bad == 0;
                }
            }
            if (lane == 0) p.need[j] = ok ? need : -1;
        }
    }
    exchange(nct);
    // offsets of the entries (every CTA scans the whole list and keeps those its warps will serve), and the free list
    int total_need = 0;
    for (int j0 = 0; j0 < p.n; j0 += kPlanThreads) {
        const int j = j0 + tid;
        const int v = j < p.n ? max(__ldcg(p.need + j), 0) : 0;
        int total;
        const int before = block_scan(v, &total);
        if (j < p.n && (few ? j % kAll / kPlanThreads : j % kAllWarps / kPlanWarps) == rank) p.offs[j] = total_need + before;
        total_need += total;
    }
    int before;
    const int total_free = slice_total(p.counts, gwarp, kAllWarps, &before);
    if (total_need > 0 && before < total_need && mine > 0) {
        int at = before;
        walk_refs(p.refs, lo, hi, [&](int i, const int (&r)[4], int k) {
            int c = 0;
            for (int j = 0; j < 4; ++j) c += j < k && r[j] == 0;
            int w = at + lanes_before(c);
            at += warp_total(c);
            for (int j = 0; j < 4; ++j)
                if (j < k && r[j] == 0) {
                    if (w < total_need) p.free_list[w] = i + j;
                    ++w;
                }
        });
    }
    if (gtid == 0 && total_need > total_free) report(p.status, MSK_ERR_CAPACITY, kWhere | 4, total_need, total_free);
    exchange(nct);
    if (few) {
        for (int j = gtid; j < p.n; j += kAll) {
            const int need = __ldcg(p.need + j), off = __ldcg(p.offs + j);
            if (need <= 0) continue;
            if (kFork) {
                const bool got = off < total_free;
                const int page = got ? __ldcg(p.free_list + off) : -1;
                p.ops[j].y = page;
                if (got) p.refs[page] = 1;
                else p.ops[j].w = 2;
            } else {
                const int row = p.list[j], seq = p.seq_lens[row];
                int* held = p.page_table + static_cast<size_t>(row) * p.max_pages;
                const int last = min(static_cast<int>((static_cast<long long>(seq) + p.q_len - 1) >> p.page_log), p.max_pages - 1);
                int k = off;
                for (int lp = seq >> p.page_log; lp <= last; ++lp) {
                    if (held[lp] >= 0) continue;
                    if (k < total_free) {
                        const int page = __ldcg(p.free_list + k);
                        held[lp] = page;
                        p.refs[page] = 1;
                    }
                    ++k;
                }
            }
        }
        if (kFork || p.cache_loc == nullptr) return;
        exchange(nct);
        for (int t = gtid; t < p.tokens; t += kAll) {  // a thread per token
            const int j = t / p.q_len, row = p.list[j];
            long long loc = -1;
            if (__ldcg(p.need + j) >= 0) {
                const long long pos = static_cast<long long>(p.seq_lens[row]) + (t - j * p.q_len), lp = pos >> p.page_log;
                const int page = lp < p.max_pages ? __ldcg(p.page_table + static_cast<size_t>(row) * p.max_pages + lp) : -1;
                if (page >= 0) loc = (static_cast<long long>(page) << p.page_log) + (pos & (p.page_size - 1));
            }
            p.cache_loc[t] = loc;
        }
        return;
    }
    if constexpr (!kFork) {
        for (int j = gwarp; j < p.n; j += kAllWarps) {
            const int need = __ldcg(p.need + j), off = __ldcg(p.offs + j), row = p.list[j];
            int n_tok, first_loc;
            tokens_of(p, j, &n_tok, &first_loc);
            const int seq = need >= 0 ? p.seq_lens[row] : 0;
            int* held = need >= 0 ? p.page_table + static_cast<size_t>(row) * p.max_pages : nullptr;
            if (need > 0) {
                const int first = seq >> p.page_log;
                const int last = min(static_cast<int>((static_cast<long long>(seq) + n_tok - 1) >> p.page_log), p.max_pages - 1);
                int at = off;
                for (int lp0 = first; lp0 <= last; lp0 += 32) {
                    const int lp = lp0 + lane;
                    const bool want = lp <= last && held[lp] < 0;
                    const uint32_t all = __ballot_sync(0xffffffffu, want);
                    const int k = at + __popc(all & ((1u << lane) - 1u));
                    if (want && k < total_free) {
                        const int page = __ldcg(p.free_list + k);
                        held[lp] = page;
                        p.refs[page] = 1;
                    }
                    at += __popc(all);
                }
                __syncwarp();
            }
            if (p.cache_loc != nullptr) {
                for (int t = lane; t < n_tok; t += 32) {
                    const long long pos = static_cast<long long>(seq) + t;
                    const int page = held != nullptr && (pos >> p.page_log) < p.max_pages ? held[pos >> p.page_log] : -1;
                    p.cache_loc[static_cast<long long>(first_loc) + t] =
                        page >= 0 ? (static_cast<long long>(page) << p.page_log) + (pos & (p.page_size - 1)) : -1;
                }
            }
        }
    }
}

// Entries of the listed rows go back: all of them (free) or those wholly before the window and behind the sinks (trim).
__global__ void __launch_bounds__(256) pages_drop_kernel(PlanArgs p, int blocks_per_row, int window, int sinks, int trim) {
    pdl_wait();
    pdl_launch_dependents();
    const int j = blockIdx.x / blocks_per_row, part = blockIdx.x % blocks_per_row;
    const int row = p.list[j];
    if (row < 0 || row >= p.rows) {
        if (part == 0 && threadIdx.x == 0) report(p.status, MSK_ERR_BOUNDS, kWhere | 5, row, p.rows);
        return;
    }
    int first = 0, last = p.max_pages;
    if (trim) {
        // the next token, at position seq, sees what lies behind seq - window: pages that end there or earlier go
        const long long low = static_cast<long long>(p.seq_lens[row]) - window + 1;
        first = static_cast<int>((static_cast<long long>(sinks) + p.page_size - 1) >> p.page_log);
        last = low > 0 ? static_cast<int>(min(low >> p.page_log, static_cast<long long>(p.max_pages))) : 0;
    }
    for (int lp = first + part * 256 + static_cast<int>(threadIdx.x); lp < last; lp += blocks_per_row * 256) {
        int* e = p.page_table + static_cast<size_t>(row) * p.max_pages + lp;
        if (*e >= 0) {
            const int id = atomicExch(e, -1);  // a row that is listed twice gives its pages back once
            if (id >= p.num_pages) report(p.status, MSK_ERR_BOUNDS, kWhere | 6, id, p.num_pages);
            else if (id >= 0) atomicSub(p.refs + id, 1);
        }
    }
    if (!trim && part == 0 && threadIdx.x == 0) p.seq_lens[row] = 0;
}

// `bytes` (a multiple of 16) from src to dst by one CTA, in flight kCopyChunk at a time.
__device__ __forceinline__ void copy_chunk(uint8_t* dst, const uint8_t* src, int bytes) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int at = (u * kCopyThreads + static_cast<int>(threadIdx.x)) * 16;
        if (at < bytes) v[u] = __ldcs(reinterpret_cast<const uint4*>(src + at));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int at = (u * kCopyThreads + static_cast<int>(threadIdx.x)) * 16;
        if (at < bytes) __stcs(reinterpret_cast<uint4*>(dst + at), v[u]);
    }
}

// Fork, second launch: the children's table rows, the shared pages' counts, and the data of the pages that are copied.
// CTAs [0, row_blocks) do the rows, the others the data.
__global__ void __launch_bounds__(kCopyThreads) pages_fork_kernel(PlanArgs p, Caches caches, int row_blocks, int blocks_per_row) {
    pdl_wait();
    pdl_launch_dependents();
    if (static_cast<int>(blockIdx.x) < row_blocks) {
        const int j = blockIdx.x / blocks_per_row, part = blockIdx.x % blocks_per_row;
        const int4 op = __ldcg(p.ops + j);
        if (op.w == 0) return;
        const int child = p.list[j], par = p.parents[j];
        const int seq = p.seq_lens[par], full = seq >> p.page_log;
        for (int lp = part * kCopyThreads + static_cast<int>(threadIdx.x); lp < p.max_pages; lp += blocks_per_row * kCopyThreads) {
            int* e = p.page_table + static_cast<size_t>(child) * p.max_pages + lp;
            const int old = *e;
            int id = -1;
            if (op.w == 1) id = lp < full ? p.page_table[static_cast<size_t>(par) * p.max_pages + lp] : lp == full ? op.y : -1;
            if (id >= p.num_pages) {
                report(p.status, MSK_ERR_BOUNDS, kWhere | 6, id, p.num_pages);
                id = -1;
            }
            *e = id;
            if (id >= 0 && lp < full) atomicAdd(p.refs + id, 1);
            if (old >= 0 && old < p.num_pages) atomicSub(p.refs + old, 1);  // what the child's row held before
        }
        if (part == 0 && threadIdx.x == 0) p.seq_lens[child] = op.w == 1 ? seq : 0;
        return;
    }
    const int page_bytes = p.page_size * caches.token_bytes;
    const int chunks = (page_bytes + kCopyChunk - 1) / kCopyChunk;
    const long long units = static_cast<long long>(p.n) * caches.n * chunks;
    for (long long u = blockIdx.x - row_blocks; u < units; u += gridDim.x - row_blocks) {
        const int c = static_cast<int>(u % chunks), k = static_cast<int>(u / chunks % caches.n);
        const int4 op = __ldcg(p.ops + u / chunks / caches.n);
        const int bytes = op.z * caches.token_bytes - c * kCopyChunk;
        if (op.w != 1 || op.y < 0 || bytes <= 0) continue;
        const size_t at = static_cast<size_t>(c) * kCopyChunk;
        copy_chunk(caches.p[k] + static_cast<size_t>(op.y) * page_bytes + at, caches.p[k] + static_cast<size_t>(op.x) * page_bytes + at,
                   min(bytes, kCopyChunk));
    }
}

// Compact, first launch: with n pages in use, the k-th page in use from n on goes to the k-th free page below n.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(PlanArgs p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, nct = gridDim.x;
    const int gtid = rank * kPlanThreads + tid, gwarp = rank * kPlanWarps + warp;
    const int kAll = nct * kPlanThreads, kAllWarps = nct * kPlanWarps;
    int *c_live = p.counts, *c_hole = c_live + kCluster * kPlanWarps, *c_move = c_hole + kCluster * kPlanWarps, *result = c_move + kCluster * kPlanWarps;
    pdl_wait();
    pdl_launch_dependents();
    int lo, hi;
    slice_of(p, gwarp, kAllWarps, &lo, &hi);
    int mine = 0, before;
    walk_refs(p.refs, lo, hi, [&](int, const int (&r)[4], int k) {
        for (int j = 0; j < 4; ++j) mine += j < k && r[j] > 0;
    });
    mine = warp_total(mine);
    if (lane == 0) c_live[gwarp] = mine;
    exchange(nct);
    const int live = slice_total(c_live, gwarp, kAllWarps, &before);
    // a page below `live` that is free, or one in use from `live` on: as many of the one as of the other
    auto kind = [&](int page, int r) { return page < live ? (r <= 0 ? 1 : 0) : (r > 0 ? 2 : 0); };
    int holes = 0, moves = 0;
    walk_refs(p.refs, lo, hi, [&](int i, const int (&r)[4], int k) {
        for (int j = 0; j < 4; ++j) {
            const int t = j < k ? kind(i + j, r[j]) : 0;
            holes += t == 1, moves += t == 2;
        }
    });
    holes = warp_total(holes), moves = warp_total(moves);
    if (lane == 0) c_hole[gwarp] = holes, c_move[gwarp] = moves;
    exchange(nct);
    int hole_at, move_at;
    slice_total(c_hole, gwarp, kAllWarps, &hole_at);
    const int all_moves = slice_total(c_move, gwarp, kAllWarps, &move_at);
    if (holes + moves > 0) {
        walk_refs(p.refs, lo, hi, [&](int i, const int (&r)[4], int k) {
            int nh = 0, nm = 0;
            for (int j = 0; j < 4; ++j) {
                const int t = j < k ? kind(i + j, r[j]) : 0;
                nh += t == 1, nm += t == 2;
            }
            const int both = lanes_before(nh | nm << 16);  // at most 128 of either in a step
            int wh = hole_at + (both & 0xffff), wm = move_at + (both >> 16);
            hole_at += warp_total(nh), move_at += warp_total(nm);
            for (int j = 0; j < 4; ++j) {
                const int t = j < k ? kind(i + j, r[j]) : 0;
                if (t == 1) p.dst[wh++] = i + j;
                if (t == 2) p.src[wm++] = i + j;
            }
        });
    }
    exchange(nct);
    for (int k = gtid; k < all_moves; k += kAll) {
        const int s = __ldcg(p.src + k), d = __ldcg(p.dst + k);
        p.remap[s] = d;
        p.refs[d] = __ldcg(p.refs + s);
        p.refs[s] = 0;
    }
    if (gtid == 0) {
        result[0] = live, result[1] = all_moves;
        if (p.result != nullptr) p.result[0] = live, p.result[1] = all_moves;
    }
}

// Compact, second launch: the table's entries, then the pages' data.
__global__ void __launch_bounds__(kCopyThreads) pages_compact_kernel(PlanArgs p, Caches caches) {
    pdl_wait();
    pdl_launch_dependents();
    const int* result = p.counts + 3 * kCluster * kPlanWarps;
    const int live = __ldcg(result), moves = __ldcg(result + 1);
    if (moves == 0) return;
    const long long entries = static_cast<long long>(p.rows) * p.max_pages;
    for (long long i = static_cast<long long>(blockIdx.x) * kCopyThreads + threadIdx.x; i < entries; i += static_cast<long long>(gridDim.x) * kCopyThreads) {
        const int id = p.page_table[i];
        if (id >= live && id < p.num_pages) p.page_table[i] = __ldcg(p.remap + id);
    }
    const int page_bytes = p.page_size * caches.token_bytes;
    const int chunks = (page_bytes + kCopyChunk - 1) / kCopyChunk;
    const long long units = static_cast<long long>(moves) * caches.n * chunks;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int c = static_cast<int>(u % chunks), k = static_cast<int>(u / chunks % caches.n);
        const long long i = u / chunks / caches.n;
        const size_t at = static_cast<size_t>(c) * kCopyChunk;
        copy_chunk(caches.p[k] + static_cast<size_t>(__ldcg(p.dst + i)) * page_bytes + at,
                   caches.p[k] + static_cast<size_t>(__ldcg(p.src + i)) * page_bytes + at, min(page_bytes - static_cast<int>(at), kCopyChunk));
    }
}

size_t up256(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

// Workspace: counts | claim, is_parent [rows] | need, offs [n] | ops [n] | three lists of pages
size_t layout(const MskPages* q, int n, uint8_t* ws, PlanArgs* a) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = ws + at;
        at += up256(bytes);
        return p;
    };
    int* counts = reinterpret_cast<int*>(take((3 * kCluster * kPlanWarps + 4) * 4));
    int* claim = reinterpret_cast<int*>(take(static_cast<size_t>(q->rows) * 4));
    int* is_parent = reinterpret_cast<int*>(take(static_cast<size_t>(q->rows) * 4));
    int* need = reinterpret_cast<int*>(take(static_cast<size_t>(n) * 4));
    int* offs = reinterpret_cast<int*>(take(static_cast<size_t>(n) * 4));
    int4* ops = reinterpret_cast<int4*>(take(static_cast<size_t>(n) * 16));
    int* src = reinterpret_cast<int*>(take(static_cast<size_t>(q->num_pages) * 4));
    int* dst = reinterpret_cast<int*>(take(static_cast<size_t>(q->num_pages) * 4));
    int* remap = reinterpret_cast<int*>(take(static_cast<size_t>(q->num_pages) * 4));
    if (a != nullptr) {
        a->counts = counts, a->claim = claim, a->is_parent = is_parent, a->need = need, a->offs = offs, a->ops = ops;
        a->src = src, a->dst = dst, a->remap = remap, a->free_list = src;
    }
    return at;
}

int fill(const MskPages* q, const int* list, int n, void* scratch, size_t bytes, bool workspace, int* status, PlanArgs* a) {
    if (q == nullptr || !q->page_table || !q->seq_lens || !q->refs || n < 0 || (n > 0 && list == nullptr)) return MSK_ERR_INVALID;
    if (q->rows < 1 || q->max_pages < 1 || q->num_pages < 1) return MSK_ERR_UNSUPPORTED;
    if (q->page_size < 1 || (q->page_size & (q->page_size - 1)) != 0) return MSK_ERR_UNSUPPORTED;
    *a = PlanArgs{};
    a->page_table = q->page_table, a->seq_lens = q->seq_lens, a->refs = q->refs;
    a->rows = q->rows, a->max_pages = q->max_pages, a->num_pages = q->num_pages, a->page_size = q->page_size;
    while ((1 << a->page_log) < q->page_size) ++a->page_log;
    a->list = list, a->n = n, a->status = status;
    if (workspace) {
        if (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 255) != 0) return MSK_ERR_INVALID;
        if (layout(q, n, static_cast<uint8_t*>(scratch), a) > bytes) return MSK_ERR_INVALID;
    }
    return 0;
}

int fill_caches(const MskPages* q, void* const* caches, int n_caches, int token_bytes, Caches* c) {
    if (n_caches < 0 || n_caches > kMaxCaches || (n_caches > 0 && caches == nullptr)) return MSK_ERR_INVALID;
    if (token_bytes < 16 || token_bytes % 16 != 0 || static_cast<long long>(token_bytes) * q->page_size > (1 << 30)) return MSK_ERR_UNSUPPORTED;
    *c = Caches{};
    c->n = n_caches, c->token_bytes = token_bytes;
    for (int i = 0; i < n_caches; ++i) {
        if (caches[i] == nullptr || (reinterpret_cast<uintptr_t>(caches[i]) & 15) != 0) return MSK_ERR_INVALID;
        c->p[i] = static_cast<uint8_t*>(caches[i]);
    }
    return 0;
}

template <class... Params, class... Args>
int launch(void (*kernel)(Params...), unsigned grid, unsigned block, bool chained, unsigned cluster, void* stream, Args... args) {
    cudaLaunchAttribute attr[2];
    int n = 0;
    cudaLaunchConfig_t cfg = {};
    if (chained) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(block), cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr, cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : MSK_ERR_CUDA;
}

// A planning kernel: one CTA, or one cluster of eight where there is much to rank or to look up.
template <class... Params>
int launch_plan(void (*kernel)(Params...), const PlanArgs& a, void* stream) {
    const unsigned n = a.num_pages > kOneCta || a.n > 1024 ? kCluster : 1;
    return launch(kernel, n, kPlanThreads, false, n, stream, a);
}

// CTAs for page data: enough to fill every SM, no more than there are pieces.
unsigned copy_ctas(long long units) {
    const long long most = 148 * 8;
    return static_cast<unsigned>(units < 1 ? 1 : units < most ? units : most);
}

int drop(const MskPages* q, const int* rows, int n, int window, int sinks, int trim, int* status, void* stream) {
    PlanArgs a;
    const int rc = fill(q, rows, n, nullptr, 0, false, status, &a);
    if (rc != 0 || n == 0) return rc;
    const int per_row = (q->max_pages + 1023) / 1024;
    if (static_cast<long long>(n) * per_row > 0x7fffffffll) return MSK_ERR_UNSUPPORTED;
    return launch(pages_drop_kernel, static_cast<unsigned>(n) * per_row, 256, false, 1, stream, a, per_row, window, sinks, trim);
}

}  // namespace
}  // namespace msk

extern "C" int msk_pages_scratch_bytes(const MskPages* q, int n, size_t* bytes) {
    if (q == nullptr || bytes == nullptr || n < 0 || q->rows < 1 || q->num_pages < 1) return MSK_ERR_INVALID;
    *bytes = msk::layout(q, n, nullptr, nullptr);
    return 0;
}

extern "C" int msk_pages_free(const MskPages* q, const int32_t* rows, int n, int* status, void* stream) {
    return msk::drop(q, rows, n, 0, 0, 0, status, stream);
}

extern "C" int msk_pages_trim(const MskPages* q, const int32_t* rows, int n, int window, int sinks, int* status, void* stream) {
    if (window < 0 || sinks < 0) return MSK_ERR_INVALID;
    if (window == 0) n = 0;  // every position stays visible: nothing to give back
    return msk::drop(q, rows, n, window, sinks, 1, status, stream);
}

extern "C" int msk_pages_extend(const MskPages* q, const int32_t* rows, int n, int q_len, const int32_t* cu_seqlens, int tokens,
                                int64_t* cache_loc, void* scratch, size_t scratch_bytes, int* status, void* stream) {
    using namespace msk;
    PlanArgs a;
    const int rc = fill(q, rows, n, scratch, scratch_bytes, n > 0, status, &a);
    if (rc != 0) return rc;
    if (cu_seqlens == nullptr && (q_len < 0 || static_cast<long long>(n) * q_len > 0x7fffffffll)) return MSK_ERR_INVALID;
    if (cu_seqlens != nullptr && tokens < 0) return MSK_ERR_INVALID;
    if (n == 0) return 0;
    a.q_len = q_len, a.cu = cu_seqlens, a.tokens = cu_seqlens != nullptr ? tokens : n * q_len;
    a.cache_loc = reinterpret_cast<long long*>(cache_loc);
    return launch_plan(pages_plan_kernel<false>, a, stream);
}

extern "C" int msk_pages_fork(const MskPages* q, const int32_t* parents, const int32_t* children, int n, void* const* caches, int n_caches,
                              int token_bytes, void* scratch, size_t scratch_bytes, int* status, void* stream) {
    using namespace msk;
    PlanArgs a;
    int rc = fill(q, children, n, scratch, scratch_bytes, n > 0, status, &a);
    if (rc != 0) return rc;
    Caches c;
    rc = fill_caches(q, caches, n_caches, token_bytes, &c);
    if (rc != 0 || n == 0) return rc;
    if (parents == nullptr) return MSK_ERR_INVALID;
    a.parents = parents;
    const int per_row = (q->max_pages + 4 * kCopyThreads - 1) / (4 * kCopyThreads);
    const long long row_blocks = static_cast<long long>(n) * per_row;
    const long long chunks = (static_cast<long long>(q->page_size) * token_bytes + kCopyChunk - 1) / kCopyChunk;
    const unsigned data = copy_ctas(static_cast<long long>(n) * n_caches * chunks);
    if (row_blocks + data > 0x7fffffffll) return MSK_ERR_UNSUPPORTED;
    rc = launch_plan(pages_plan_kernel<true>, a, stream);
    if (rc != 0) return rc;
    return launch(pages_fork_kernel, static_cast<unsigned>(row_blocks) + data, kCopyThreads, true, 1, stream, a, c, static_cast<int>(row_blocks), per_row);
}

extern "C" int msk_pages_compact(const MskPages* q, void* const* caches, int n_caches, int token_bytes, int32_t* result, void* scratch,
                                 size_t scratch_bytes, int* status, void* stream) {
    using namespace msk;
    PlanArgs a;
    int rc = fill(q, nullptr, 0, scratch, scratch_bytes, true, status, &a);
    if (rc != 0) return rc;
    Caches c;
    rc = fill_caches(q, caches, n_caches, token_bytes, &c);
    if (rc != 0) return rc;
    a.result = result;
    rc = launch_plan(pages_compact_plan_kernel, a, stream);
    if (rc != 0) return rc;
    const long long chunks = (static_cast<long long>(q->page_size) * token_bytes + kCopyChunk - 1) / kCopyChunk;
    const long long table = (static_cast<long long>(q->rows) * q->max_pages + kCopyThreads - 1) / kCopyThreads;
    const long long data = static_cast<long long>(q->num_pages / 2 + 1) * n_caches * chunks;  // at most half of the pages move
    return launch(pages_compact_kernel, copy_ctas(data > table ? data : table), kCopyThreads, true, 1, stream, a, c);
}
