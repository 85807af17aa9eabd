// Gated attention for prompts: any number of new tokens per request behind any number of cached ones, over the paged
// FP8-E4M3 cache, with a sliding window and first tokens that stay visible.  Two launches, three when the keys are split:
//
//   prep     one CTA per token: RMSNorm, scale and RoPE of its queries (rounded to BF16, kept as FP16 in the workspace) and
//            keys; keys and values quantised to E4M3 and written into the pages the page table names.  Keys and angles are
//            taken in 64 bits (2 us of 310 for 16 prompts of 1 to 1024 tokens).  One more CTA lists the work units (request, first token), unless
//            they are few and every CTA finds its own.  Bound by memory: 18 KB per token at 32 + 4 + 4 heads.
//   main     one CTA, or a pair of CTAs on neighbouring SMs, per (unit of 32 or 64 new tokens, KV head, split): flash
//            attention.  The 8 query heads of a KV head and the tokens together are the rows of the product: a CTA has 2
//            tiles of 128 rows = 16 tokens x 8 heads.
//   combine  one warp per (token, head): joins the splits' (m, l, O); used when there are fewer units than SMs.
//
// Main kernel, per 128-key tile (FP16 tensor-core operands: E4M3 cache values and BF16 queries are exact in FP16; FP16
// probabilities are off by 2^-12 of their value down to 2^-22 of the row's largest, below that by 2^-33 of the largest, so the
// result carries little more than its last rounding):
//   copying warp     TMA boxes of the K and V pages into E4M3 staging
//   converting warps E4M3 -> FP16 into the swizzled operand tiles, value rows no token sees as zeros
//   MMA warp         S = Q K^T into TMEM (128 x 128 FP32 per row tile), O += P V with P from TMEM
//   softmax warps    thread = row: the row's 128 scores come from TMEM in one go, no shuffles; p = 2^(s - m) goes back as
//                    FP16 over the scores.  The running reference m lies below the maximum and moves only when a score
//                    outgrows what FP16 holds, so the accumulator in TMEM is rescaled a few times per row, not per tile
//                    (800 clocks each time and the wait for the last product, in whichever warp has such a row).
// The products run ahead of the softmax in halves of 64 keys: while the softmax works on one half of a row tile's scores,
// the tensor cores add the other half's product and put the next tile's scores in its place.  (With whole tiles each tile
// waited 1300 clocks for its next scores, a third of the loop; a third row tile does not fit.)
// Values are 0 * V for the tokens that do not see them, so a NaN among them is zeroed where not all tokens of the unit see it,
// and the rows that do are made NaN at the end.
// Measured (32 + 4 heads, replayed in a graph / called from Python): 8192 tokens, full, behind nothing: 564 / 610 us = 0.97 /
// 0.90 PFLOP/s, 59 / 55 % of the rate of a BF16 matrix product; three documents of 2500 to 4099 tokens under window 1024 + 64
// sinks 345 / 347 us, 0.47 PFLOP/s of visible keys; 16 prompts of 1 to 1024 tokens under window 1024 + 4 294 / 297 us; 16 x 8
// tokens 22 / 25 us; 19 tokens behind 7001 cached ones 14.7 / 18.9 us.  No unit is near its limit (tensor cores and
// special-function units a third busy each); the time goes with the chain of the two softmax warps of each scheduler: 1750 - 1850
// clocks per 64 keys and two row tiles, of which a loop of the softmax alone (scores from TMEM, maximum, exponentials, back to
// TMEM) takes 1500 on the scheduler that also issues the products.  Per unit come 12 us: 3 until the first scores, 2 for the
// last product, 5.5 for norm, gate and stores, 1 until the next CTA runs.  Under a window a unit has only 5 to 40 tiles, so
// these and the masked parts of its edge tiles weigh more.  Small calls: prep 3 us, main from 6, combine 1, and 1.5 us between the
// launches.
// Tried without gain: an MMA warp per row tile, a reference without a maximum, turn-taking softmax warps, scores fetched a
// half ahead, a persistent grid, output tiles stored by TMA, four softmax warpgroups, more polynomials; for units with one
// row tile, half of each tile's keys for each group of softmax warps (16 x 8 tokens: 22.6 us).
// TMEM: S (P over the first half of each half) and O, 128 columns each, for two row tiles = all 512 columns.
// Pairs (CG = 2, tcgen05 cta_group::2): a tile's products run over both SMs, 256 rows, each CTA bringing its rows and half of
// the K and V tile.  A single CTA is bound by shared memory: per tile 128 KB of Q and K reads, 64 KB of V, 96 KB of
// conversion and 32 KB of TMA writes take 2560 clocks at 128 bytes each, the products 2048; a pair's CTA moves 192 KB.
#include "attn_common.cuh"
#include "msk.h"
#include "ptx.cuh"
#include "tmap.cuh"

namespace msk {
namespace {

constexpr int kTile = 128;                  // keys per tile
constexpr int kTok = 16;                    // tokens per row tile
constexpr int kThreads = 512;               // softmax A | softmax B | converting | MMA, copying, one that waits for the queries, one that checks the lists
constexpr int kQBytes = 32768;              // one row tile of queries: two swizzled halves of 64 channels
template <int CG>
struct Geo {
    static constexpr int kSlots = CG == 1 ? 2 : 3;      // FP16 operand slots, K and V each
    static constexpr int kStages = CG == 1 ? 1 : 2;     // E4M3 staging, K and V each
    static constexpr int kF16 = 32768 / CG;             // one CTA's part of a K tile (keys) or V tile (channels) as FP16
    static constexpr int kF8 = 16384 / CG;
    static constexpr int kKeys = kTile / CG;            // K rows here
    static constexpr int kChan = 128 / CG;              // V channels here
    // Half a tile's scores: 64 columns.  Of a pair, each CTA brings 32 keys: columns 0 .. 31 are keys 32 half .. , columns
    // 32 .. 63 the keys 64 further.  A single CTA takes 64 keys in a row.
    static constexpr int kHalf = 64 / CG;               // keys between the first columns of the two halves
    static constexpr int kNext = 32 * CG;               // keys between column 0 and column 32
    static constexpr int kSmem = 2 * kQBytes + 2 * kSlots * kF16 + 2 * kStages * kF8 + 1024;
};
static_assert(Geo<1>::kSmem <= 231000 && Geo<2>::kSmem <= 231000, "shared memory");
constexpr float kNegRef = -1.0e30f;
constexpr int kPolyEvery = 4;               // of the pairs of probabilities, every how manieth goes to the FMA pipe
constexpr float kLazy = 15.75f;             // how far (in powers of two) a score may lie above its row's reference
constexpr float kBelow = 2.0f;              // how far a new reference lies below the row's maximum: this and log2 of the key tiles,
constexpr float kMostBelow = 13.0f;         // at most this
constexpr int kMaxUnitsHeader = 4;          // ints before the unit list: their number, padding
constexpr int kBuckets = 256;

struct PromptArgs {
    const __nv_bfloat16* qkv;
    int ld_qkv;
    __nv_bfloat16* out;
    int ld_out;
    uint8_t* k_cache;
    uint8_t* v_cache;
    const float* k_scale;
    const float* v_scale;
    const int* seq_lens;
    const int* cu;    // or NULL: q_len tokens each
    int q_len;
    const int* page_table;
    int max_pages;
    const float* inv_freq;
    int B, T, Hq, Hkv, page_size, page_log, num_pages, window, sinks, splits, max_units;
    int last_tile;    // of the page table
    int out_wide;     // rows of out allow 32-byte stores
    float qk_scale_factor, q_scale, s_scale;  // queries are stored times q_scale (a power of two); scores times s_scale * k_scale
    __half* q16;      // [T, Hq, 128]
    int* units;       // [kMaxUnitsHeader + 4 * max_units]: request, first row of qkv, tokens, first position
    int unit;         // tokens per unit
    int direct;       // the main kernel finds its unit itself (few requests, one wave: the order does not matter)
    float* part_o;    // [splits, T * Hq, 128]
    float* part_ml;   // [splits, T * Hq, 2]
    int* status;
};

__device__ __forceinline__ int first_row(const PromptArgs& p, int b) {  // of qkv and out; b = B: the end
    return p.cu != nullptr ? min(max(p.cu[b], 0), p.T) : b * p.q_len;
}
__device__ __forceinline__ int new_tokens(const PromptArgs& p, int b) { return max(first_row(p, b + 1) - first_row(p, b), 0); }

// RMSNorm (weightless, eps 1e-5), scale and interleaved RoPE of one 128-wide head row, 4 values per lane.
__device__ __forceinline__ void norm_turn(float (&x)[4], float post_scale, const float (&c)[2], const float (&s)[2], bool turn) {
    float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
    ss = warp_sum(ss);
    const float r = 1.0f / sqrtf(ss * (1.0f / 128.0f) + 1e-5f);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (x[i] * r) * post_scale;
    if (turn) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float e = x[2 * h], o = x[2 * h + 1];
            x[2 * h] = e * c[h] - o * s[h];
            x[2 * h + 1] = e * s[h] + o * c[h];
        }
    }
}

// How many key tiles a unit's tokens see, and where they are: [0, sink_tiles) and [first, first + tiles - sink_tiles).  None lie
// behind the page table's last one, whatever seq_lens says (the prep kernel reports it).
__device__ __forceinline__ int key_tiles(const PromptArgs& p, int p_first, int p_last, int* first, int* sink_tiles) {
    const int W = p.window, snk = W > 0 ? p.sinks : 0;
    *first = (W > 0 && p_first >= W ? p_first - W + 1 : 0) / kTile;
    const int last = min(p_last / kTile, p.last_tile);
    *sink_tiles = min(min(snk / kTile + (snk % kTile != 0), *first), last + 1);
    return last - *first + 1 + *sink_tiles;
}

// The unit list: each request's new tokens in groups of p.unit, the units with the most key tiles first (a counting sort over
// the number of tiles), so that the last units to start are short.  One CTA of 256 threads: a warp per request, a lane per
// unit.  The order inside a bucket is left to the atomics; no unit's result depends on it.
__device__ void list_units(const PromptArgs& p) {
    __shared__ int hist[kBuckets], n_s[256], seq_s[256], row_s[256], sum_s[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    hist[tid] = 0;
    int total = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int b0 = 0; b0 < p.B; b0 += 256) {
            __syncthreads();
            const int b = b0 + tid;
            if (b < p.B) n_s[tid] = new_tokens(p, b), seq_s[tid] = p.seq_lens[b], row_s[tid] = first_row(p, b);
            __syncthreads();
            for (int r = warp; r < 256 && b0 + r < p.B; r += 8) {
                const int n = n_s[r], units = (n + p.unit - 1) / p.unit;
                for (int i = lane; i < units; i += 32) {
                    const int n_tok = min(n - i * p.unit, p.unit), p_first = seq_s[r] + i * p.unit;
                    int first, sink;
                    const int bucket = kBuckets - 1 - min(max(key_tiles(p, p_first, p_first + n_tok - 1, &first, &sink), 0), kBuckets - 1);
                    const int at = atomicAdd(&hist[bucket], 1);
                    if (pass == 1 && at < p.max_units)
                        *reinterpret_cast<int4*>(p.units + kMaxUnitsHeader + 4 * at) = make_int4(b0 + r, row_s[r] + i * p.unit, n_tok, p_first);
                }
            }
        }
        __syncthreads();
        if (pass == 0) {  // counts -> first places
            const int v = hist[tid];
            int inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += u;
            }
            if (lane == 31) sum_s[warp] = inc;
            __syncthreads();
            int before = 0;
            for (int w = 0; w < 8; ++w) {
                if (w < warp) before += sum_s[w];
                total += sum_s[w];
            }
            hist[tid] = before + inc - v;
        }
    }
    if (tid == 0) {
        if (total > p.max_units) report(p.status, MSK_ERR_CAPACITY, MSK_K_PROMPT << 8 | 1, total, p.max_units);
        p.units[0] = min(total, p.max_units);
    }
}

__global__ void __launch_bounds__(256) prompt_prep_kernel(PromptArgs p) {
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == 0 && !p.direct) {  // first, it takes longest
        list_units(p);
        return;
    }
    const int t = blockIdx.x - (p.direct ? 0 : 1);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // everything that needs no look-up is asked for first: the token's head rows, the frequencies, the scales
    const __nv_bfloat16* row = p.qkv + static_cast<size_t>(t) * p.ld_qkv;
    const int heads = p.Hq + 2 * p.Hkv;
    constexpr int U = 5;  // rows in flight per warp: 8 warps cover 40 heads at once
    uint2 raw[U];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h0 + 8 * u < heads) raw[u] = __ldg(reinterpret_cast<const uint2*>(row + (h0 + 8 * u) * 128 + 4 * lane));
    };
    fetch(warp);
    const bool turn = p.inv_freq != nullptr;
    const float my_freq = turn && threadIdx.x < 64 ? __ldg(p.inv_freq + threadIdx.x) : 0.0f;
    const float k_scale = __ldg(p.k_scale), v_scale = __ldg(p.v_scale);
    // the request of token t: the last b with cu[b] <= t, by steps of 32 requests
    int lo = 0, hi = p.B;  // cu[lo] <= t < cu[hi] is looked for in [lo, hi)
    if (p.cu == nullptr) lo = t / p.q_len, hi = lo + 1;
    else if (t >= p.cu[p.B] || t < p.cu[0]) return;  // a row behind the last sequence
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + step * lane;
        const bool le = at < hi && p.cu[at] <= t;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
        const int nlo = lo + step * k;
        hi = min(hi, nlo + step);
        lo = nlo;
    }
    const int b = lo;
    const int pos = p.seq_lens[b] + t - (p.cu != nullptr ? p.cu[b] : b * p.q_len);
    // cos and sin of the token's 64 angles, in 64 bits (a product in 32 bits is off by up to 5e-4 at position 8192)
    __shared__ double2 angles[64];
    if (turn && threadIdx.x < 64) {
        double sn, cs;
        sincos(static_cast<double>(pos) * static_cast<double>(my_freq), &sn, &cs);
        angles[threadIdx.x] = make_double2(cs, sn);
    }
    const int page = pos >> p.page_log;
    const int id = pos >= 0 && page < p.max_pages ? p.page_table[static_cast<size_t>(b) * p.max_pages + page] : -1;
    const bool page_ok = id >= 0 && id < p.num_pages;
    if (!page_ok && threadIdx.x == 0) report(p.status, MSK_ERR_BOUNDS, MSK_K_PROMPT << 8 | 2, id, page);
    const size_t slot = page_ok ? (static_cast<size_t>(id) << p.page_log) + (pos & (p.page_size - 1)) : 0;
    __syncthreads();
    double2 turn2[2] = {make_double2(1.0, 0.0), make_double2(1.0, 0.0)};
    if (turn) turn2[0] = angles[2 * lane], turn2[1] = angles[2 * lane + 1];
    const float c[2] = {static_cast<float>(turn2[0].x), static_cast<float>(turn2[1].x)};
    const float s[2] = {static_cast<float>(turn2[0].y), static_cast<float>(turn2[1].y)};
    for (int h0 = warp; h0 < heads; h0 += 8 * U) {
        if (h0 != warp) fetch(h0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + 8 * u;
            if (h >= heads) break;
            float x[4] = {bf16lo(raw[u].x), bf16hi(raw[u].x), bf16lo(raw[u].y), bf16hi(raw[u].y)};
            if (h < p.Hq) {
                norm_turn(x, p.qk_scale_factor, c, s, turn);
                __half2 a[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    a[i] = __floats2half2_rn(__bfloat162float(__float2bfloat16(x[2 * i])) * p.q_scale,
                                             __bfloat162float(__float2bfloat16(x[2 * i + 1])) * p.q_scale);
                *reinterpret_cast<uint2*>(p.q16 + (static_cast<size_t>(t) * p.Hq + h) * 128 + 4 * lane) =
                    make_uint2(*reinterpret_cast<uint32_t*>(&a[0]), *reinterpret_cast<uint32_t*>(&a[1]));
            } else {
                const bool key = h < p.Hq + p.Hkv;
                if (key) {
                    // in 64 bits up to the quantisation: in 32 a few bytes of a million fall to the other side of a rounding
                    // border, 6 % off
                    const double a[4] = {x[0], x[1], x[2], x[3]};
                    double ss = a[0] * a[0] + a[1] * a[1] + a[2] * a[2] + a[3] * a[3];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const double r = 1.0 / (sqrt(ss * (1.0 / 128.0) + 1e-5) * static_cast<double>(k_scale));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[2 * i] = static_cast<float>((a[2 * i] * turn2[i].x - a[2 * i + 1] * turn2[i].y) * r);
                        x[2 * i + 1] = static_cast<float>((a[2 * i] * turn2[i].y + a[2 * i + 1] * turn2[i].x) * r);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = __fdiv_rn(x[i], v_scale);
                }
                const uint32_t w = f2_to_e4m3x2(x[0], x[1]) | f2_to_e4m3x2(x[2], x[3]) << 16;
                const int kv = h - p.Hq - (key ? 0 : p.Hkv);
                if (page_ok)
                    *reinterpret_cast<uint32_t*>((key ? p.k_cache : p.v_cache) + (slot * p.Hkv + kv) * 128 + 4 * lane) = w;
            }
        }
    }
}

__device__ __forceinline__ uint32_t low_bits(int n) {  // bits [0, n) set, n clamped to [0, 32]
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

// 32 bytes to one address: a full sector per lane.
__device__ __forceinline__ void store32(void* dst, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

template <int CG>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, PromptArgs p) {
    using G = Geo<CG>;
    constexpr int NS = G::kSlots, SS = G::kStages;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[4 * SS + 4 * NS + 14];
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t spoilt[2];  // one bit per token of the unit: it sees a NaN value at a position others do not see

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = CG == 1 ? 0 : static_cast<int>(cluster_ctarank());  // which half of the pair; the even one issues the MMAs
    const int unit_id = blockIdx.x / CG;
    const int h = unit_id % p.Hkv, sp = (unit_id / p.Hkv) % p.splits, slot_u = unit_id / (p.Hkv * p.splits);
    const int where = MSK_K_PROMPT << 8;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t s_q = base, s_k = s_q + 2 * kQBytes, s_v = s_k + NS * G::kF16, s_f8 = s_v + NS * G::kF16;
    uint8_t* g_k = gbase + 2 * kQBytes;
    uint8_t* g_v = g_k + NS * G::kF16;
    uint8_t* g_f8 = g_v + NS * G::kF16;
    auto bar = [&](int i) { return smem_u32(&bars[i]); };
    // staging full / free, K stages then V stages; operand slots full / free, K then V; queries; output; halves of the
    // scores and of P per row tile; products added per row tile.  With a pair, "full", "queries" and "P" collect both CTAs' arrivals at the even CTA;
    // what the MMAs signal arrives in both.
    const uint32_t st_full = bar(0), st_free = bar(2 * SS), op_full = bar(4 * SS), op_free = bar(4 * SS + 2 * NS),
                   q_here = bar(4 * SS + 4 * NS), q_full = q_here + 8, o_done = q_here + 16, s_done = q_here + 32, p_ready = q_here + 64,
                   pv_done = q_here + 96;
    auto arrive_issuer = [&](uint32_t b) {
        if constexpr (CG == 1) mbar_arrive(b);
        else mbar_arrive_cluster(dsmem_addr(b, 0));
    };

    if (tid == 32) {
        for (int i = 0; i < 2 * SS; ++i) mbar_init(st_full + 8 * i, 1), mbar_init(st_free + 8 * i, 4);
        for (int i = 0; i < 2 * NS; ++i) mbar_init(op_full + 8 * i, 4 * CG), mbar_init(op_free + 8 * i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(o_done + 8 * i, 1), mbar_init(pv_done + 8 * i, 1);
        for (int i = 0; i < 4; ++i) mbar_init(s_done + 8 * i, 1), mbar_init(p_ready + 8 * i, 4 * CG);
        mbar_init(q_here, 1);
        mbar_init(q_full, CG);
        spoilt[0] = spoilt[1] = 0;
        fence_mbar_init();
    }
    if (tid == 64) prefetch_tmap(&tm_q), prefetch_tmap(&tm_k), prefetch_tmap(&tm_v);
    if (warp == 0) tmem_alloc_cg<CG>(smem_u32(&tmem_slot), 512);
    // Where a CTA finds its unit itself, only the copying warp waits for the prep kernel, with the first tiles of old keys on
    // their way: what came before the prep kernel is complete (it waits for that before it lets this one start).
    if (!p.direct) pdl_wait();
    pdl_launch_dependents();

    // ---------------- this CTA's unit: the pair's row tile g covers tokens 16 CG g .. of the unit, this CTA 16 of them
    int4 u = make_int4(0, 0, 0, 0);  // request, first row, tokens, first position
    int old_end = 0;                 // positions below are older than this call (known to direct units)
    if (!p.direct) {
        const int n_units = __ldcg(p.units);
        if (slot_u < n_units) u = __ldcg(reinterpret_cast<const int4*>(p.units + kMaxUnitsHeader + 4 * slot_u));
    } else if (p.cu == nullptr) {
        const int per_req = (p.q_len + p.unit - 1) / p.unit, rb = slot_u / per_req, at = (slot_u - rb * per_req) * p.unit;
        if (rb < p.B) {
            old_end = p.seq_lens[rb];
            u = make_int4(rb, rb * p.q_len + at, min(p.q_len - at, p.unit), old_end + at);
        }
    } else {  // a lane per request (B <= 32): which one's groups of tokens hold number slot_u
        const int n = lane < p.B ? new_tokens(p, lane) : 0, row0 = lane < p.B ? first_row(p, lane) : 0, seq = lane < p.B ? p.seq_lens[lane] : 0;
        const int groups = (n + p.unit - 1) / p.unit;
        int inc = groups;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, inc > slot_u);
        if (behind != 0) {
            const int src = __ffs(behind) - 1;
            const int at = (slot_u - (__shfl_sync(0xffffffffu, inc, src) - __shfl_sync(0xffffffffu, groups, src))) * p.unit;
            old_end = __shfl_sync(0xffffffffu, seq, src);
            u = make_int4(src, __shfl_sync(0xffffffffu, row0, src) + at, min(__shfl_sync(0xffffffffu, n, src) - at, p.unit), old_end + at);
        }
    }
    const int b = u.x, tok0 = u.y, n_tok = u.z, p_first = u.w, p_last = p_first + max(n_tok, 1) - 1;
    const int W = p.window, snk = W > 0 ? p.sinks : 0;
    int t_first, sink_tiles;
    const int tiles = key_tiles(p, p_first, p_last, &t_first, &sink_tiles);
    const int win_tiles = tiles - sink_tiles;  // these first: their many keys set the references that the sinks' few would set too low
    const int per = (tiles + p.splits - 1) / p.splits;
    const int v_begin = sp * per;
    const int nt = n_tok > 0 ? max(0, min(per, tiles - v_begin)) : 0;
    const bool two = n_tok > kTok * CG;                    // the second row tile has tokens
    auto base_of = [&](int i) { return (v_begin + i + (v_begin + i < win_tiles ? t_first : -win_tiles)) * kTile; };
    auto tok_of = [&](int g) { return kTok * (CG * g + rank); };  // first token of row tile g here, within the unit

    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 1) __syncthreads();
    else cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp < 8) {
        // ================ softmax: thread = row of row tile g
        const float k_scale = __ldg(p.k_scale), v_scale = __ldg(p.v_scale);
        const int g = warp >> 2, row = tid & 127, j = tok_of(g) + (row >> 3), head = h * 8 + (row & 7);
        const int pos = p_first + j;
        const bool live = j < n_tok;
        const size_t token = static_cast<size_t>(tok0) + j;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + g * 128, t_o = tmem + lanes + 256 + g * 128;
        const float scale = k_scale * p.s_scale;
        const int g_first = p_first + tok_of(g), g_last = g_first + kTok - 1;
        const float below = fminf(kBelow + __log2f(static_cast<float>(max(tiles, 1))), kMostBelow);
        float m = kNegRef, top = kNegRef, l = 0.0f;  // reference, maximum, sum
        bool ok = true;
        if ((g == 0 || two) && nt > 0) {
            for (int t = 0; t < 2 * nt; ++t) {  // 64 keys at a time
                const int half = t & 1, par = (t >> 1) & 1;
                const uint32_t t_x = t_s + 64 * half;
                ok = mbar_wait(s_done + 16 * g + 8 * half, par, p.status, where | 3) && ok;
                tc_fence_after();
                uint32_t x[2][32];
                float mx[4];
#pragma unroll
                for (int c = 0; c < 2; ++c) tmem_ld32(t_x + 32 * c, x[c]);
                tmem_wait_ld();
                const int s0 = base_of(t >> 1) + G::kHalf * half;  // position of the first key; the second 32 lie kNext further
                if (s0 + G::kNext + 31 > g_first || (W > 0 && s0 <= g_last - W && s0 + G::kNext + 32 > snk)) {
                    // an edge of what the rows see: one bit per key
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = s0 + G::kNext * c;
                        uint32_t vis = low_bits(pos - at + 1);
                        if (W > 0) vis &= ~low_bits(pos - W - at + 1) | low_bits(snk - at);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(vis & (1u << e))) x[c][e] = 0xff800000u;  // -inf
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    auto v = [&](int e) { return __uint_as_float(x[c >> 1][16 * (c & 1) + e]); };
                    mx[c] = max3(v(0), v(1), v(2));
#pragma unroll
                    for (int e = 3; e < 15; e += 2) mx[c] = max3(mx[c], v(e), v(e + 1));
                    mx[c] = fmaxf(mx[c], v(15));
                }
                // A new reference lies 2^below below the row's maximum and serves until a score lies 2^kLazy above it: the row's
                // largest p is between the two, and FP16's rounding at its small end, 2^-25, times the number of keys is 2^-20 of
                // the largest weight at any length (from 262144 keys on more).  That much, because thousands of keys may lie
                // 2^-20 below one that draws the weight and still carry the output, when that one's value is small.  (References
                // 2^4 above the maximum lost such keys, up to 9.7 % of a row of 8192, and saved moves: 8192 tokens full 585 us
                // against 608, three documents under a window 333 and 347, 16 mixed prompts 286 and 298.  Moving to the half
                // tile's maximum instead of the row's costs as much again.)
                const float tops = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale;
                top = fmaxf(top, tops);
                // Rows behind the unit's last token (the next request's, or a padding row's leftovers) move nothing: the bits of
                // a request are its own.
                const bool move = live && tops - m > kLazy;
                if (__any_sync(0xffffffffu, move)) {
                    // all of the warp's rows move up, not only those that must: four sinks first leave 32 low references, and
                    // one of the rows outgrew its own in most of the following steps
                    const float m_new = fmaxf(m, top - below);
                    const float alpha = ex2(m - m_new);
                    m = m_new;
                    l *= alpha;
                    if (t > 0) {  // the accumulator follows, once the last product has been added
                        ok = mbar_wait(pv_done + 8 * g, (t - 1) & 1, p.status, where | 2) && ok;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(t_o + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st16(t_o + c, o);
                        }
                    }
                }
                const float2 scale2 = make_float2(scale, scale), off2 = make_float2(-m, -m);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                uint32_t w[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const int cc = e >> 4, k = 2 * (e & 15);
                    const float2 y = fma2(make_float2(__uint_as_float(x[cc][k]), __uint_as_float(x[cc][k + 1])), scale2, off2);
                    const float2 v = e % kPolyEvery == kPolyEvery - 1 ? ex2_poly2(y) : make_float2(ex2(y.x), ex2(y.y));
                    sum[e & 1] = add2(sum[e & 1], v);
                    w[e] = pack_half(v.x, v.y);
                }
                tmem_st32(t_x, w);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_issuer(p_ready + 16 * g + 8 * half);
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
            }
            // ---- the row's end: value = o * v_scale / l, RMSNorm over 128 channels, sigmoid gate, BF16 (or the split's part)
            uint4 gate[16];
            if (p.splits == 1 && live) {  // asked for before the last product is done
                const uint4* src = reinterpret_cast<const uint4*>(p.qkv + token * p.ld_qkv + (p.Hq + 2 * p.Hkv + head) * 128);
#pragma unroll
                for (int e = 0; e < 16; ++e) gate[e] = __ldg(src + e);
            }
            ok = mbar_wait<0, (CG > 1)>(o_done + 8 * g, 0, p.status, where | 4) && ok;
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            // one NaN channel makes the row's norm, and so the row, NaN
            if (live && (*static_cast<volatile uint32_t*>(&spoilt[j >> 5]) >> (j & 31) & 1)) l = __int_as_float(0x7fffffff);
            if (p.splits == 1) {
                const float inv = v_scale / l;
                float ss = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32(t_o + 32 * c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float o = __uint_as_float(v[e]) * inv;
                        ss = fmaf(o, o, ss);
                    }
                }
                const float r = inv / sqrtf(ss * (1.0f / 128.0f) + 1e-5f);
                __nv_bfloat16* dst = p.out + token * p.ld_out + head * 128;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t v[16];
                    tmem_ld16(t_o + 16 * c, v);
                    tmem_wait_ld();
                    if (live && ok) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint4 q = gate[2 * c + (e >> 2)];
                            const uint32_t gw = (e & 3) == 0 ? q.x : (e & 3) == 1 ? q.y : (e & 3) == 2 ? q.z : q.w;
                            const float a = __fdividef(__uint_as_float(v[2 * e]) * r, 1.0f + __expf(-bf16lo(gw)));
                            const float d = __fdividef(__uint_as_float(v[2 * e + 1]) * r, 1.0f + __expf(-bf16hi(gw)));
                            w[e] = pack_bf16(a, d);
                        }
                        if (p.out_wide) {
                            store32(dst + 16 * c, w);
                        } else {
                            reinterpret_cast<uint4*>(dst)[2 * c] = make_uint4(w[0], w[1], w[2], w[3]);
                            reinterpret_cast<uint4*>(dst)[2 * c + 1] = make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    }
                }
            } else {
                const size_t r = (static_cast<size_t>(sp) * p.T + token) * p.Hq + head;
                if (live) *reinterpret_cast<float2*>(p.part_ml + 2 * r) = make_float2(ok ? m : kNegRef, ok ? l : 0.0f);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld32(t_o + 32 * c, v);
                    tmem_wait_ld();
                    if (live) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            const uint32_t w[8] = {v[e], v[e + 1], v[e + 2], v[e + 3], v[e + 4], v[e + 5], v[e + 6], v[e + 7]};
                            store32(p.part_o + r * 128 + 32 * c + e, w);
                        }
                    }
                }
            }
        } else if (p.splits > 1 && live) {  // a split without keys
            const size_t r = (static_cast<size_t>(sp) * p.T + token) * p.Hq + head;
            *reinterpret_cast<float2*>(p.part_ml + 2 * r) = make_float2(kNegRef, 0.0f);
        }
    } else if (warp < 12) {
        // ================ converting: E4M3 staging -> FP16 operand tiles (this CTA's half of the keys of K, of the channels of V)
        const int w = warp - 8;
        bool ok = true;
        int stage = 0, st_ph = 0, slot = 0, op_ph = 0;
        for (int i = 0; i < nt && ok; ++i) {
            const int s0 = base_of(i);
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
                ok = mbar_wait(st_full + 8 * (kv * SS + stage), st_ph, p.status, where | 5) && ok;
                if (i >= NS) ok = mbar_wait(op_free + 8 * (kv * NS + slot), op_ph ^ 1, p.status, where | 6) && ok;
                if (!ok) break;
                const uint8_t* src = g_f8 + (kv * SS + stage) * G::kF8;
                uint8_t* dst = (kv ? g_v : g_k) + slot * G::kF16;
                // All loads before the first store: the compiler does not move a load over a store to shared memory, and a
                // tile took 1150 clocks of load latencies instead of 400.
                constexpr int U = 8 / CG;
                uint4 in[U];
                int rr[U], cc[U];  // row of the tile and 16-byte piece of the row (V of a pair: rows of 64 bytes)
                if (CG == 2 && kv) {
                    // 8 lanes: two rows of 64 contiguous bytes
#pragma unroll
                    for (int e = 0; e < U; ++e) {
                        rr[e] = w * 32 + e * 8 + (lane >> 2);
                        cc[e] = lane & 3;
                        in[e] = *reinterpret_cast<const uint4*>(src + rr[e] * 64 + cc[e] * 16);
                    }
                } else {
                    // 8 lanes: 64 bytes of row r and the other 64 of row r + 1: no conflicts in loads or stores
                    constexpr int kRows = G::kKeys / 4;  // rows of K per warp
                    const int rows = kv ? 32 : kRows;
#pragma unroll
                    for (int e = 0; e < U; ++e) {
                        rr[e] = w * rows + (e >> 1) * 8 + (lane >> 2);
                        cc[e] = (lane & 3) + 4 * (((lane >> 2) ^ e) & 1);
                        in[e] = *reinterpret_cast<const uint4*>(src + rr[e] * 128 + cc[e] * 16);
                    }
                }
                if (kv && (s0 + kTile - 1 > p_first || (W > 0 && s0 <= p_last - W && s0 + kTile > snk))) {
                    // Positions that not all tokens of the unit see.  What none sees may be anything: zeros, so that 0 * V
                    // stays 0.  A NaN that some see must not reach the others by 0 * V either: zeros, and a note to those.
                    uint32_t notes = 0;
                    auto seen = [&](int pos, int* from, int* to) {  // tokens [from, to) of the unit see position pos
                        *from = max(pos - p_first, 0);
                        *to = W > 0 && pos >= snk && pos - p_first < n_tok - W ? pos - p_first + W : n_tok;
                    };
#pragma unroll
                    for (int e = 0; e < U; ++e) {
                        int from, to;
                        seen(s0 + rr[e], &from, &to);
                        const bool none = from >= to, bad = !none && to - from < n_tok && has_nan(in[e]);
                        if (none || bad) in[e] = make_uint4(0, 0, 0, 0);
                        notes |= bad ? 1u << e : 0u;
                    }
                    if (notes != 0) {
#pragma unroll 1
                        for (int e = 0; e < U; ++e) {
                            if (!(notes >> e & 1)) continue;
                            int from, to;
                            seen(s0 + w * 32 + (CG == 2 ? e : e >> 1) * 8 + (lane >> 2), &from, &to);
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t who = low_bits(to - 32 * c) & ~low_bits(from - 32 * c);
                                atomicOr(&spoilt[c], who);
                                if constexpr (CG == 2) dsmem_or_b32(dsmem_addr(smem_u32(&spoilt[c]), rank ^ 1), who);
                            }
                        }
                        if (CG == 2) __threadfence();  // before the arrival at the even CTA, which releases at CTA scope
                    }
                }
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    const uint32_t q[4] = {in[e].x, in[e].y, in[e].z, in[e].w};
                    uint32_t o[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q[k]), __NV_E4M3);
                        const __half2_raw d = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(q[k] >> 16), __NV_E4M3);
                        o[2 * k] = *reinterpret_cast<const uint32_t*>(&a);
                        o[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&d);
                    }
                    // 64 channels per swizzled row of 128 bytes; the second 64 behind all rows of the first
                    uint8_t* half = dst + (cc[e] >> 2) * (kv ? 16384 : G::kKeys * 128);
                    *reinterpret_cast<uint4*>(half + swz128(rr[e], (cc[e] & 3) * 32)) = make_uint4(o[0], o[1], o[2], o[3]);
                    *reinterpret_cast<uint4*>(half + swz128(rr[e], (cc[e] & 3) * 32 + 16)) = make_uint4(o[4], o[5], o[6], o[7]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(st_free + 8 * (kv * SS + stage));
                    arrive_issuer(op_full + 8 * (kv * NS + slot));
                }
            }
            if (++stage == SS) stage = 0, st_ph ^= 1;
            if (++slot == NS) slot = 0, op_ph ^= 1;
        }
    } else {
        if (warp == 12) {
            // ================ the MMA warp: all lanes run the loop, one issues (of a pair, the even CTA's)
            if (nt > 0 && rank == 0) {
                const uint32_t leader = elect_one();
                const uint32_t id_qk = umma_idesc(128 * CG, 64, 0, 0, 0, 0), id_pv = umma_idesc(128 * CG, 128, 0, 0, 0, 1);
                const uint64_t d_q = umma_smem_desc(s_q, 16, 1024, kSwizzle128), d_k = umma_smem_desc(s_k, 16, 1024, kSwizzle128);
                const uint64_t d_v = umma_smem_desc(s_v, 16384, 1024, kSwizzle128);
                auto wait = [&](uint32_t b, int parity, int site) { return mbar_wait<0, (CG > 1)>(b, parity, p.status, where | site); };
                auto scores = [&](int g, int slot, int half) {  // 64 keys' S_g = Q_g K^T
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t oq = ((e >> 2) * 16384 + (e & 3) * 32) >> 4, ok_ = ((e >> 2) * (G::kKeys * 128) + (e & 3) * 32) >> 4;
                        umma_f16_ss_if<CG>(leader, tmem + g * 128 + 64 * half, d_q + (g * kQBytes >> 4) + oq,
                                           d_k + ((slot * G::kF16 + half * G::kHalf * 128) >> 4) + ok_, id_qk, e != 0);
                    }
                    umma_commit_if<CG>(leader, s_done + 16 * g + 8 * half);
                };
                auto output = [&](int g, int slot, int half, bool first) {  // O_g (+)= P_g V over those 64 keys
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = half * G::kHalf + (e >> 1) * G::kNext + (e & 1) * 16;
                        umma_f16_ts_if<CG>(leader, tmem + 256 + g * 128, tmem + g * 128 + 64 * half + 8 * e, d_v + ((slot * G::kF16 + row * 128) >> 4),
                                           id_pv, !first || e != 0);
                    }
                    umma_commit_if<CG>(leader, pv_done + 8 * g);
                };
                bool ok = wait(q_full, 0, 7) && wait(op_full, 0, 8);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        scores(0, 0, half);
                        if (two) scores(1, 0, half);
                    }
                    umma_commit_if<CG>(leader, op_free);
                }
                int slot = 0, ph = 0;
                for (int i = 0; i < nt && ok; ++i) {
                    const bool more = i + 1 < nt;
                    const int nslot = slot + 1 == NS ? 0 : slot + 1, nph = slot + 1 == NS ? ph ^ 1 : ph;
                    ok = wait(op_full + 8 * (NS + slot), ph, 9);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            if (g == 1 && !two) break;
                            ok = ok && wait(p_ready + 16 * g + 8 * half, i & 1, 10 + g);
                            if (!ok) break;
                            tc_fence_after();
                            output(g, slot, half, i == 0 && half == 0);
                            if (more) {  // the next tile's scores over the probabilities just read
                                if (half == 0 && g == 0) {
                                    ok = wait(op_full + 8 * nslot, nph, 12);
                                    if (!ok) break;
                                    tc_fence_after();
                                }
                                scores(g, nslot, half);
                            }
                        }
                    }
                    if (!ok) break;
                    umma_commit_if<CG>(leader, op_free + 8 * (NS + slot));
                    if (more) umma_commit_if<CG>(leader, op_free + 8 * nslot);
                    slot = nslot, ph = nph;
                }
                umma_commit_if<CG>(leader, o_done);
                umma_commit_if<CG>(leader, o_done + 8);
            }
            __syncwarp();
        } else if (warp == 13 && nt > 0) {
            // ================ the copying warp
            const int ppt = kTile >> p.page_log;  // pages per tile, <= 16: lane j fetches page j
            auto page_of = [&](int i) {
                const int pg = (base_of(i) >> p.page_log) + lane;
                int id = lane < ppt && pg < p.max_pages ? p.page_table[static_cast<size_t>(b) * p.max_pages + pg] : -1;
                if (id >= p.num_pages || id < -1) {
                    report(p.status, MSK_ERR_BOUNDS, where | 13, id, p.num_pages);
                    id = -1;
                }
                return id;  // -1: zeros
            };
            // of a pair, K pages: the keys [64 rank, 64 rank + 64) of the tile; a page of 128 keys is split
            const int key0 = lane << p.page_log;
            const bool k_mine = lane < ppt && (CG == 1 || p.page_size == kTile || (key0 >= rank * G::kKeys && key0 < (rank + 1) * G::kKeys));
            const int k_in_page = CG == 2 && p.page_size == kTile ? rank * G::kKeys : 0;
            const uint32_t k_at = CG == 2 ? (p.page_size == kTile ? 0 : key0 - rank * G::kKeys) * 128 : key0 * 128;
            auto fetch = [&](int kv, int stage, int id) {
                const uint32_t full = st_full + 8 * (kv * SS + stage), dst = s_f8 + (kv * SS + stage) * G::kF8;
                if (lane == 0) mbar_expect_tx(full, G::kF8);
                __syncwarp();
                if (kv == 0) {
                    if (k_mine) tma_load_4d(dst + k_at, &tm_k, full, 0, h, k_in_page, id);
                } else {
                    if (lane < ppt) tma_load_4d(dst + key0 * G::kChan, &tm_v, full, CG == 2 ? rank * G::kChan : 0, h, 0, id);
                }
            };
            int id = page_of(0), i = 0;
            bool ok = true;
            int stage = 0, ph = 0;
            if (p.direct) {
                for (; i < SS && i < nt && base_of(i) + kTile <= old_end; ++i) {
                    const int next = i + 1 < nt ? page_of(i + 1) : -1;
                    fetch(0, stage, id);
                    fetch(1, stage, id);
                    id = next;
                    if (++stage == SS) stage = 0, ph ^= 1;
                }
                pdl_wait();
            }
            if (lane == 0) {
                mbar_expect_tx(q_here, (two ? 2 : 1) * kQBytes);
                for (int g = 0; g < (two ? 2 : 1); ++g)
                    for (int c = 0; c < 2; ++c)
                        tma_load_3d(s_q + g * kQBytes + c * 16384, &tm_q, q_here, 64 * c, h * 8, tok0 + tok_of(g));
            }
            for (; i < nt && ok; ++i) {
                const int next = i + 1 < nt ? page_of(i + 1) : -1;
                for (int kv = 0; kv < 2; ++kv) {
                    if (i >= SS) ok = mbar_wait(st_free + 8 * (kv * SS + stage), ph ^ 1, p.status, where | 14) && ok;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    fetch(kv, stage, id);
                }
                id = next;
                if (++stage == SS) stage = 0, ph ^= 1;
            }
            __syncwarp();
        } else if (warp == 13) {
            if (p.direct) pdl_wait();  // no CTA ends before the prep kernel does
        } else if (warp == 14 && nt > 0) {
            // ================ this CTA's queries have arrived: tell the MMA warp
            const bool ok = mbar_wait(q_here, 0, p.status, where | 15);
            if (lane == 0 && ok) arrive_issuer(q_full);
            __syncwarp();
        } else if (warp == 15 && blockIdx.x == 0 && p.cu != nullptr) {
            // ================ the spare warp of the first CTA: requests that name rows which are not there
            for (int r = lane; r < p.B; r += 32) {
                const int from = p.cu[r], to = p.cu[r + 1];
                if (from < 0 || to < from || to > p.T) report(p.status, MSK_ERR_BOUNDS, where | 16, to, p.T);
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncwarp();
    if constexpr (CG == 1) __syncthreads();
    else cluster_sync_all();  // nothing of this CTA's memory is needed by its pair any more
    if (warp == 0) tmem_dealloc_cg<CG>(tmem, 512);
}

// Joins the splits of one (token, head) per warp: lane = 4 channels of the output, and one or two splits' (m, l).  Everything is
// asked for at once: with the loads one behind the other
// 19 tokens behind 7001 (6 splits) took 18.2 us, now 15.8.
__global__ void __launch_bounds__(256) prompt_combine_kernel(PromptArgs p) {
    const int lane = threadIdx.x & 31;
    const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int token = static_cast<int>(row / p.Hq), head = static_cast<int>(row % p.Hq);
    const uint2 g = __ldg(reinterpret_cast<const uint2*>(p.qkv + static_cast<size_t>(token) * p.ld_qkv + (p.Hq + 2 * p.Hkv + head) * 128 + 4 * lane));
    const float v_scale = __ldg(p.v_scale);
    const bool mine = token < first_row(p, p.B) && token >= first_row(p, 0);  // a row of some request
    pdl_wait();
    pdl_launch_dependents();
    const size_t stride = static_cast<size_t>(p.T) * p.Hq;
    float2 ml[2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
        ml[c] = lane + 32 * c < p.splits ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * ((lane + 32 * c) * stride + row))) : make_float2(kNegRef, 0.0f);
    constexpr int U = 8;
    float4 v[U];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < p.splits) v[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((s0 + u) * stride + row) * 128 + 4 * lane));
    };
    fetch(0);
    float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float w[2], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 2; ++c) w[c] = ml[c].y != 0.0f ? ex2(ml[c].x - m) : 0.0f;  // a split without keys has no weight; NaN counts
    const float l = warp_sum(w[0] * ml[0].y + w[1] * ml[1].y);
    for (int s0 = 0; s0 < p.splits; s0 += U) {
        if (s0 > 0) fetch(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float ws = __shfl_sync(0xffffffffu, s0 + u < 32 ? w[0] : w[1], (s0 + u) & 31);
            if (s0 + u < p.splits && ws != 0.0f) o[0] += ws * v[u].x, o[1] += ws * v[u].y, o[2] += ws * v[u].z, o[3] += ws * v[u].w;
        }
    }
    const float inv = l != 0.0f ? v_scale / l : 0.0f;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= inv, ss += o[i] * o[i];
    ss = warp_sum(ss);
    const float r = 1.0f / sqrtf(ss * (1.0f / 128.0f) + 1e-5f);
    const float gate[4] = {bf16lo(g.x), bf16hi(g.x), bf16lo(g.y), bf16hi(g.y)};
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * r / (1.0f + __expf(-gate[i]));
    if (mine)
        *reinterpret_cast<uint2*>(p.out + static_cast<size_t>(token) * p.ld_out + head * 128 + 4 * lane) =
            make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
}

struct Plan {
    int max_units, splits, cg;
    size_t q16, units, ml, o, total;  // byte offsets, and the end
};

int plan_prompt(const MskPromptParams* q, Plan* plan) {
    if (q->d != 128 || q->Hkv < 1 || q->Hq != 8 * q->Hkv || q->B < 1 || q->T < 1 || q->max_pages < 1) return MSK_ERR_UNSUPPORTED;
    if (q->page_size < 8 || q->page_size > 128 || (q->page_size & (q->page_size - 1)) != 0) return MSK_ERR_UNSUPPORTED;
    if (q->window < 0 || q->sinks < 0 || q->splits < 0 || q->splits > 64) return MSK_ERR_INVALID;
    // Pairs of CTAs where requests bring more than 32 tokens on average: a unit of 64 tokens then fills both.
    plan->cg = static_cast<long long>(q->T) > 32ll * q->B ? 2 : 1;
    const int unit = 2 * kTok * plan->cg;
    const long long units = q->cu_seqlens_q == nullptr && q->q_len > 0
                                ? static_cast<long long>(q->B) * ((q->q_len + unit - 1) / unit)
                                : static_cast<long long>(q->T) / unit + q->B;  // sum of ceil(n / unit) is at most this
    plan->max_units = static_cast<int>(units < q->T ? units : q->T);
    long long tiles = (static_cast<long long>(q->max_pages) * q->page_size + kTile - 1) / kTile;
    if (q->window > 0) {
        const long long w = (static_cast<long long>(q->window) + unit) / kTile + 2 + (static_cast<long long>(q->sinks) + kTile - 1) / kTile;
        if (w < tiles) tiles = w;
    }
    plan->splits = q->splits;
    if (q->splits == 0) {
        // Fewer units than SMs: the keys are split into pieces of equal tiles, as many as find an SM, down to one tile.  Parts
        // cost their way through memory, a tile's time for some 3500 rows (token, head): 300 tokens x 32 heads over 3 tiles take
        // 21.0 us whole and 22.3 in three pieces, over 5 tiles 24.8 and 24.0; 8 tokens over 5 tiles 14.9 and 11.1.
        const long long ctas = static_cast<long long>(plan->max_units) * q->Hkv * plan->cg;
        long long most = 148 / ctas;
        if (most > 32) most = 32;
        plan->splits = 1;
        if (most > 1) {
            const long long per = (tiles + most - 1) / most;
            if ((tiles - per) * 3500 > static_cast<long long>(q->T) * q->Hq) plan->splits = static_cast<int>((tiles + per - 1) / per);
        }
    }
    auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    const size_t rows = static_cast<size_t>(q->T) * q->Hq;
    plan->q16 = 0;
    plan->units = up(rows * 256);
    plan->ml = plan->units + up((kMaxUnitsHeader + 4 * static_cast<size_t>(plan->max_units)) * 4);
    const size_t parts = plan->splits > 1 ? static_cast<size_t>(plan->splits) * rows : 0;
    plan->o = plan->ml + up(parts * 8);
    plan->total = plan->o + up(parts * 512);
    return 0;
}

}  // namespace
}  // namespace msk

extern "C" int msk_attn_prompt_scratch_bytes(const MskPromptParams* q, size_t* bytes) {
    msk::Plan plan;
    if (q == nullptr || bytes == nullptr) return MSK_ERR_INVALID;
    const int rc = msk::plan_prompt(q, &plan);
    if (rc == 0) *bytes = plan.total;
    return rc;
}

extern "C" int msk_attn_prompt(const MskPromptParams* q, int* status, void* stream) {
    using namespace msk;
    if (q == nullptr || !q->qkv || !q->out || !q->k_cache || !q->v_cache || !q->k_scale || !q->v_scale || !q->seq_lens ||
        !q->page_table || !q->scratch)
        return MSK_ERR_INVALID;
    if (q->cu_seqlens_q == nullptr && (q->q_len < 1 || static_cast<long long>(q->B) * q->q_len != q->T)) return MSK_ERR_INVALID;
    Plan plan;
    int rc = plan_prompt(q, &plan);
    if (rc != 0) return rc;
    const int wide = (2 * q->Hq + 2 * q->Hkv) * 128;
    if (q->scratch_bytes < plan.total || (reinterpret_cast<uintptr_t>(q->scratch) & 255) != 0) return MSK_ERR_INVALID;
    if (q->ld_qkv < wide || q->ld_out < q->Hq * 128 || q->ld_qkv % 8 != 0 || q->ld_out % 8 != 0) return MSK_ERR_INVALID;
    if (((reinterpret_cast<uintptr_t>(q->qkv) | reinterpret_cast<uintptr_t>(q->out) | reinterpret_cast<uintptr_t>(q->k_cache) |
          reinterpret_cast<uintptr_t>(q->v_cache)) & 15) != 0)
        return MSK_ERR_INVALID;
    if (!(q->sm_scale > 0.0f) || !(q->sm_scale < 1e30f)) return MSK_ERR_INVALID;
    const long long ctas = static_cast<long long>(plan.max_units) * plan.splits * q->Hkv * plan.cg;
    if (ctas > 0x7fffffffll || static_cast<long long>(q->T) * q->Hq > 0x7fffffffll) return MSK_ERR_UNSUPPORTED;

    uint8_t* ws = static_cast<uint8_t*>(q->scratch);
    PromptArgs a{};
    a.qkv = static_cast<const __nv_bfloat16*>(q->qkv), a.ld_qkv = q->ld_qkv;
    a.out = static_cast<__nv_bfloat16*>(q->out), a.ld_out = q->ld_out;
    a.k_cache = static_cast<uint8_t*>(q->k_cache), a.v_cache = static_cast<uint8_t*>(q->v_cache);
    a.k_scale = q->k_scale, a.v_scale = q->v_scale, a.seq_lens = q->seq_lens, a.cu = q->cu_seqlens_q, a.q_len = q->q_len;
    a.page_table = q->page_table, a.max_pages = q->max_pages, a.inv_freq = q->inv_freq;
    a.B = q->B, a.T = q->T, a.Hq = q->Hq, a.Hkv = q->Hkv, a.page_size = q->page_size, a.num_pages = q->num_pages;
    while ((1 << a.page_log) < q->page_size) ++a.page_log;
    a.last_tile = static_cast<int>((static_cast<long long>(q->max_pages) * q->page_size - 1) / kTile);
    a.window = q->window, a.sinks = q->sinks, a.splits = plan.splits, a.max_units = plan.max_units, a.unit = 2 * kTok * plan.cg;
    a.out_wide = ((reinterpret_cast<uintptr_t>(q->out) | static_cast<uintptr_t>(q->ld_out) * 2) & 31) == 0;
    a.qk_scale_factor = q->qk_scale_factor;
    // the largest power of two that keeps |q| * scale below 2^15 (|q| <= qk_scale_factor * sqrt(128) after RMSNorm)
    float qs = 1.0f;
    const float qmax = fabsf(q->qk_scale_factor) * 11.3137085f;
    while (qs * 2.0f * qmax <= 32768.0f && qs < 65536.0f) qs *= 2.0f;
    while (qs * qmax > 32768.0f && qs > 1.0f / 65536.0f) qs *= 0.5f;
    a.q_scale = qs, a.s_scale = q->sm_scale * 1.4426950408889634f / qs;
    a.direct = ctas <= 148 && (q->cu_seqlens_q == nullptr || q->B <= 32);
    a.q16 = reinterpret_cast<__half*>(ws + plan.q16), a.units = reinterpret_cast<int*>(ws + plan.units);
    a.part_ml = reinterpret_cast<float*>(ws + plan.ml), a.part_o = reinterpret_cast<float*>(ws + plan.o);
    a.status = status;

    CUtensorMap tm_q, tm_k, tm_v;
    {
        const uint64_t dims[3] = {128, static_cast<uint64_t>(q->Hq), static_cast<uint64_t>(q->T)};
        const uint64_t strides[2] = {256, static_cast<uint64_t>(q->Hq) * 256};
        const uint32_t box[3] = {64, 8, kTok};
        rc = make_tmap(&tm_q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.q16, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
        if (rc != 0) return rc;
    }
    {
        const uint64_t dims[4] = {128, static_cast<uint64_t>(q->Hkv), static_cast<uint64_t>(q->page_size), static_cast<uint64_t>(q->num_pages)};
        const uint64_t strides[3] = {128, static_cast<uint64_t>(q->Hkv) * 128, static_cast<uint64_t>(q->Hkv) * 128 * q->page_size};
        // a pair's CTA copies half of the keys of K (at most 64 rows of a page) and half of the channels of V
        const uint32_t size = static_cast<uint32_t>(q->page_size);
        const uint32_t box_k[4] = {128, 1, plan.cg == 2 && size == kTile ? size / 2 : size, 1}, box_v[4] = {128u / plan.cg, 1, size, 1};
        rc = make_tmap(&tm_k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, q->k_cache, dims, strides, box_k, CU_TENSOR_MAP_SWIZZLE_NONE);
        if (rc == 0) rc = make_tmap(&tm_v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, q->v_cache, dims, strides, box_v, CU_TENSOR_MAP_SWIZZLE_NONE);
        if (rc != 0) return rc;
    }
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MSK_ERR_CUDA;
    static bool configured[64] = {};  // per device, like the attribute itself
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(prompt_attn_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<1>::kSmem) != cudaSuccess ||
            cudaFuncSetAttribute(prompt_attn_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<2>::kSmem) != cudaSuccess)
            return MSK_ERR_CUDA;
        configured[dev] = true;
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.cg, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = attr;
    cfg.gridDim = dim3(q->T + (a.direct ? 0 : 1)), cfg.blockDim = dim3(256), cfg.numAttrs = q->pdl ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, prompt_prep_kernel, a) != cudaSuccess) return MSK_ERR_CUDA;
    cfg.gridDim = dim3(static_cast<unsigned>(ctas)), cfg.blockDim = dim3(kThreads), cfg.numAttrs = 2;
    cfg.dynamicSmemBytes = plan.cg == 2 ? Geo<2>::kSmem : Geo<1>::kSmem;
    if (cudaLaunchKernelEx(&cfg, plan.cg == 2 ? prompt_attn_kernel<2> : prompt_attn_kernel<1>, tm_q, tm_k, tm_v, a) != cudaSuccess) return MSK_ERR_CUDA;
    cfg.numAttrs = 1;
    if (plan.splits > 1) {
        cfg.gridDim = dim3(static_cast<unsigned>((static_cast<long long>(q->T) * q->Hq + 7) / 8)), cfg.blockDim = dim3(256), cfg.dynamicSmemBytes = 0;
        if (cudaLaunchKernelEx(&cfg, prompt_combine_kernel, a) != cudaSuccess) return MSK_ERR_CUDA;
    }
    return 0;
}
