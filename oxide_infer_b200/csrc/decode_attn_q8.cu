// Split-KV decode attention over the 8-bit paged cache, with a sliding window and sinks.
//
//   x_t = q.(kc_t ks_t) / sqrt(128),   o = sum_t e^{x_t} vs_t vc_t / sum_t e^{x_t}
// kc, vc codes, ks, vs the scales of the token's block.  Codes (int8 and e4m3) are exact in f16, so the products
// run on f16 tensor-core fragments of the codes themselves and the scales stay in f32:
//   w_t = 2^(x_t log2e + log2 vs_t - m)   is the weight of vc_t in the numerator (m: running maximum of the exponent,
//                                         so w stays below 2^9 whatever the scales are),
//   sum_t w_t / vs_t                      is the denominator in the same units: one multiplication per thread and stage.
// A V scale below 2^-40 counts as 2^-40 (Q8_V_SCALE_MIN_LOG2).
//
// Work decomposition, claiming, merge and failure paths are those of decode_attn.cu: items are fixed ranges of
// CHUNK keys of the row's own view (a row's arithmetic does not depend on the batch), 148 persistent CTAs claim
// them, one producer warp streams stages of 64 keys with 8 KB bulk copies through a three-stage ring.  What differs:
//
// * The view is a list of aligned groups of 16 tokens (RowView), so a copy never straddles pages and all keys of a
//   group share their scales.  (Groups of 8 tokens: a copy costs the producer about 87 clocks to issue, 16 copies and
//   the bookkeeping of a stage took it longer than the memory needs for the stage.)
// * The products are transposed: S^T = K Q^T and O^T = V^T P^T.  The cache is the M = 16 operand and the four
//   query heads are half of N = 8 columns: half the tensor instructions of the f16 kernel, whose M = 16 rows are a
//   quarter filled - this kernel has to digest twice the keys per second.
// * An m16 tile i of S^T takes its rows from the 4 groups of the stage: row r is token 4i + r/4 of group r mod 4.  ALL
//   keys of a thread therefore lie in group (lane/4) mod 4: one K scale and one V scale per thread and stage.
// * K codes go from shared memory to fragments with 16-byte loads: the order of the 128 dims inside the products is
//   permuted so that a thread's 16 consecutive bytes are its operand for four k-steps (q is loaded in the same
//   order).  Group pitch + 64 bytes: the 8 lanes of a load phase fall in distinct banks.
// * V codes are transposed by ldmatrix on pairs of dims; one byte permutation then pairs the keys, which leaves the
//   output dims of a tile in the order 0, 2, ..., 14, 1, 3, ..., 15.  Group pitch + 16 bytes (two of the 8 rows of a
//   load phase still share a bank).
// * P^T reaches its B fragment with one movmatrix per 8 keys.
// * The maximum is only raised when an exponent exceeds it by more than 8 (a factor of 256 in w, within f16's range):
//   the usual stage needs no reduction over lanes at all.
// * Consumer warp h serves KV head h.  Two warps per head (half of every group's tokens each) measured 2 us slower
//   at every size: a scheduler's two warps then wait for the same pipes in the same phases.
#include "../../include/oxi_kv.h"
#include "kernels.h"
#include "q8.cuh"

namespace oxi {

namespace dq {
constexpr int KS = 64;                            // keys per stage
constexpr int NSTAGE = 3;
constexpr uint32_t GK = 16;                       // tokens per group = per bulk copy
constexpr int NGROUP = KS / (int)GK;              // 4
constexpr int GROUP_BYTES = (int)GK * Q8_ROW_BYTES;  // 8192
constexpr int KPITCH = GROUP_BYTES + 64, VPITCH = GROUP_BYTES + 16;
constexpr int V_OFF = NGROUP * KPITCH;
constexpr int Q_OFF = V_OFF + NGROUP * VPITCH;
constexpr int Q_BYTES = NQ * HD * 2;
constexpr int DESC_OFF = Q_OFF + Q_BYTES;         // 48 bytes: row / range / flags, visible bits, page slots of the groups
constexpr int STAGE_BYTES = DESC_OFF + 64;
constexpr int CHUNK = DECODE_CHUNK;               // keys per work item (the merge's key ranges)
constexpr uint32_t CHUNK_G = CHUNK / GK;
constexpr int PAGES = 28;                         // pages of an item
static_assert(PAGES >= DECODE_PAGES, "the scales of an item's pages fit its table");
constexpr int NTABLE = 4;                         // items whose scales are in shared memory
constexpr int TABLE_BYTES = PAGES * 32;           // per page: 4 K scales, 4 V scales
constexpr int N_CONSUMER_WARPS = NKV;
constexpr int THREADS = (N_CONSUMER_WARPS + 1) * 32;
constexpr int MAX_ROWS = 1024;
constexpr size_t SMEM_BYTES = (size_t)NSTAGE * STAGE_BYTES + NTABLE * TABLE_BYTES + 4 * NSTAGE * 8 + 16 + (2 * MAX_ROWS + 1) * 4;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
static_assert(STAGE_BYTES % 16 == 0 && KPITCH % 128 == 64 && VPITCH % 128 == 16, "alignment and bank offsets");
constexpr float X_SCALE = ATTN_SCALE * LOG2E;
constexpr float RAISE = 8.0f;                     // log2 units by which exponents may exceed the maximum in use
constexpr uint32_t F_FIRST = 1u << 16, F_LAST = 1u << 17, F_END = 1u << 18;
}  // namespace dq

struct DecodeQ8Params {
    uint16_t* ctx_out;
    const uint16_t* q;
    const uint16_t* gate;  // may be null
    Q8Map map;
    const uint32_t* seq_lens;
    DecodeWorkspace ws;
    uint32_t batch, window, sinks;
    uint32_t direct;  // every row is one item, no merge follows: items in fixed order, no claims
};

// mma.m16n8k16, free to be scheduled among independent ones
__device__ __forceinline__ void mma_free(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

template <uint32_t kFmt>
__global__ void __launch_bounds__(dq::THREADS, 1)
decode_attn_q8_kernel(const DecodeQ8Params p) {
    using namespace dq;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* tables = smem + (size_t)NSTAGE * STAGE_BYTES;
    // K (with q, descriptor and scales) and V of a stage are handed over separately: a K slot is refilled while the
    // consumers are still at the stage's V
    uint64_t* k_full = reinterpret_cast<uint64_t*>(tables + NTABLE * TABLE_BYTES);
    uint64_t* v_full = k_full + NSTAGE;
    uint64_t* k_empty = v_full + NSTAGE;
    uint64_t* v_empty = k_empty + NSTAGE;
    volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(v_empty + NSTAGE);
    uint32_t* prefix = const_cast<uint32_t*>(abort_flag) + 4;
    uint32_t* s_len = prefix + MAX_ROWS + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitFault fault = p.ws.fault;
    const uint32_t wait_us = fault.skip_plus1 ? fault.limit_us : WAIT_LIMIT_US;
    uint32_t* const status = p.ws.status;
    pdl_launch_dependents();

    // ---- prologue: barriers, items per row, prefix sum (reads only the step's tables)
    if (threadIdx.x == 0) {
        for (int s = 0; s < NSTAGE; s++) {
            mbar_init(&k_full[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&k_empty[s], N_CONSUMER_WARPS);
            mbar_init(&v_empty[s], N_CONSUMER_WARPS);
        }
        *abort_flag = 0u;
        prefix[0] = 0u;
        mbar_fence_init();
    }
    for (uint32_t b = threadIdx.x; b < p.batch; b += THREADS) {
        const uint32_t slen = p.seq_lens[b];
        uint32_t n = 0;
        if (slen == 0u || slen > p.ws.max_seq_len || ((slen - 1u) >> p.map.lbs) >= p.map.max_blocks) {
            if (blockIdx.x == 0) atomicOr(status, DEV_BAD_SEQ_LEN);
        } else {
            n = row_view<GK>(slen, p.window, p.sinks).ranges(CHUNK_G);
        }
        prefix[b + 1] = n;
        s_len[b] = slen;
    }
    __syncthreads();
    if (warp == 0) {
        uint32_t carry = 0;
        for (uint32_t base = 0; base < p.batch; base += 32) {
            const uint32_t i = base + lane;
            uint32_t v = (i < p.batch) ? prefix[i + 1] : 0u;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += t;
            }
            v += carry;
            if (i < p.batch) prefix[i + 1] = v;
            carry = __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    const uint32_t total_items = prefix[p.batch];
    if (warp != N_CONSUMER_WARPS) {
        pdl_wait();  // codes, scales and q written by the preceding kernel are visible from here on
    } else {
        // =========================== producer warp ===========================
        const uint64_t policy = l2_policy_evict_first();
        const uint32_t lbs = p.map.lbs, bs_mask = (1u << lbs) - 1u;
        uint32_t fill = 0, nitem = 0;
        bool ok = true;
        // An item: row, range, and lane l's page: lanes 0 .. npa-1 hold the pages of the item's sink groups from
        // page pa on, the lanes behind them those of its window groups from page pw on.
        struct Item {
            uint32_t row, range, slen, pa, pw, npa, np, id;
        };
        auto open_item = [&](uint32_t item) -> Item {
            Item it;
            // the row: the last b with prefix[b] <= item, by two looks of the whole warp (batch <= 32 * 32)
            const uint32_t step = (p.batch + 31u) / 32u;
            const uint32_t above = __ballot_sync(0xffffffffu, (uint32_t)lane * step < p.batch && prefix[min(lane * step, p.batch)] <= item);
            const uint32_t lo0 = (31u - __clz(above)) * step;
            const uint32_t in = __ballot_sync(0xffffffffu, (uint32_t)lane < step && lo0 + lane < p.batch && prefix[min(lo0 + lane, p.batch)] <= item);
            const uint32_t lo = lo0 + 31u - __clz(in);
            it.row = lo;
            it.range = item - prefix[lo];
            it.slen = s_len[lo];
            const RowView rv = row_view<GK>(it.slen, p.window, p.sinks);
            const uint32_t v0 = it.range * CHUNK_G, v1 = rv.range_end(it.range, CHUNK_G), vw = max(v0, rv.gs);
            it.pa = (v0 * GK) >> lbs;
            it.npa = v0 < rv.gs ? (((min(v1, rv.gs) - 1u) * GK) >> lbs) - it.pa + 1u : 0u;
            it.pw = rv.token<GK>(vw) >> lbs;
            it.np = it.npa + (vw < v1 ? (rv.token<GK>(v1 - 1u) >> lbs) - it.pw + 1u : 0u);
            it.id = 0;
            if ((uint32_t)lane < it.np)
                it.id = __ldg(p.map.block_tables + (size_t)it.row * p.map.max_blocks +
                              ((uint32_t)lane < it.npa ? it.pa + lane : it.pw + lane - it.npa));
            return it;
        };
        // Order of the items: the first rounds go round the CTAs (item k of this CTA is blockIdx + k * grid), the last ones
        // are claimed from a counter, since SMs do not get equal shares of the memory bandwidth.  Under a saturated
        // memory pipe a round trip takes about as long as an item, and one that the producer had to wait for would
        // leave stages empty: `c` is streamed now, the pages of `n` and `m` after it have been requested, and a claim
        // behind them is in flight.
        const uint32_t rounds = total_items / gridDim.x;
        const uint32_t fixed = p.direct ? 0xffffffffu : rounds <= 8u ? min(rounds, 4u) : rounds - 4u;  // rounds in fixed order
        uint32_t asked = 0, claim = 0;  // items of this CTA so far, the claim in flight
        auto ask = [&]() {
            // in PTX: the compiler's warp-aggregated form of atomicAdd waits for the result at once
            if (asked >= max(fixed, 1u) && lane == 0)
                asm volatile("atom.global.add.u32 %0, [%1], 1;" : "=r"(claim) : "l"(p.ws.work_counter) : "memory");
        };
        auto answer = [&]() -> uint32_t {  // the item asked for last; total_items: none
            const uint32_t k = asked++;
            if (k < max(fixed, 1u)) return min(blockIdx.x + k * gridDim.x, total_items);
            const uint32_t i = __shfl_sync(0xffffffffu, claim, 0);
            return min(total_items, max(fixed, 1u) * gridDim.x + min(i, total_items));
        };
        Item c{}, n{}, m{};
        uint32_t cur = answer(), nxt = total_items, nxt2 = total_items;  // (the first item is in the fixed order)
        if (cur < total_items) {
            // block tables are inputs of the step: the first item's pages, and their blocks into L2, while the
            // preceding kernel drains (what it may still write there is read after the wait, and L2 has it then)
            c = open_item(cur);
            const RowView rv = row_view<GK>(c.slen, p.window, p.sinks);
            const uint32_t v = c.range * CHUNK_G + (lane & 15u), v1 = rv.range_end(c.range, CHUNK_G);
            const uint32_t tok = v < v1 ? rv.token<GK>(v) : 0u;
            const uint32_t ps = v >= v1 ? 0u : v < rv.gs ? (tok >> lbs) - c.pa : c.npa + (tok >> lbs) - c.pw;
            const uint32_t id = __shfl_sync(0xffffffffu, c.id, ps & 31u);
            if (v < v1 && (lane & 15) < NSTAGE * NGROUP && id < p.map.num_blocks) {
                const unsigned char* src = (lane >= 16 ? p.map.v_pool : p.map.k_pool) + (size_t)id * p.map.block_stride + (size_t)(tok & bs_mask) * Q8_ROW_BYTES;
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(min(GK, c.slen - tok) * Q8_ROW_BYTES) : "memory");
            }
        }
        pdl_wait();
        ask();
        if (cur < total_items) {
            nxt = answer();
            if (nxt < total_items) {
                ask();
                n = open_item(nxt);
                nxt2 = answer();
                if (nxt2 < total_items) {
                    ask();
                    m = open_item(nxt2);
                }
            }
        }
        while (cur < total_items && ok) {
            if ((uint32_t)lane < c.np && c.id >= p.map.num_blocks) {
                atomicOr(status, DEV_BAD_BLOCK);
                c.id = 0;
            }
            const uint32_t nchunks = prefix[c.row + 1] - prefix[c.row];
            const RowView rv = row_view<GK>(c.slen, p.window, p.sinks);
            const uint32_t v0 = c.range * CHUNK_G, v1 = rv.range_end(c.range, CHUNK_G);
            unsigned char* table = tables + (nitem % NTABLE) * TABLE_BYTES;
            for (uint32_t v = v0; v < v1; v += NGROUP, ++fill) {
                // Whatever does not need the slot comes before the wait for it: a slot's refill starts when its last
                // consumer lets go.  Lanes 0..3 have the K groups, lanes 4..7 the V groups, lane 8 the q row.
                const uint32_t slot = fill % NSTAGE;
                const bool first = v == v0, last = v + NGROUP >= v1;
                const uint32_t g = lane & (NGROUP - 1), vg = v + g;
                const bool live = vg < v1;
                const uint32_t tok = live ? rv.token<GK>(vg) : 0u;
                const uint32_t ps = !live ? 0u : vg < rv.gs ? (tok >> lbs) - c.pa : c.npa + (tok >> lbs) - c.pw;
                const uint32_t id = __shfl_sync(0xffffffffu, c.id, ps & 31u);
                const uint32_t nk = live ? min(GK, c.slen - tok) : 0u;
                const uint32_t vis = live ? rv.visible_bits<GK>(tok) : 0u;
                // only a row's last group is shorter than 16 tokens
                const uint32_t keys = last ? (v1 - v) * GK - (v1 == rv.ng ? (0u - c.slen) & (GK - 1u) : 0u) : (uint32_t)KS;
                const uint32_t bytes = keys * Q8_ROW_BYTES;
                const bool is_v = lane >= NGROUP;
                const unsigned char* src = (is_v ? p.map.v_pool : p.map.k_pool) + (size_t)id * p.map.block_stride + (size_t)(tok & bs_mask) * Q8_ROW_BYTES;
                unsigned char* sb = smem + (size_t)slot * STAGE_BYTES;
                const uint32_t sbase = smem_u32(sb), dst = sbase + (is_v ? V_OFF + g * VPITCH : g * KPITCH);
                const uint32_t parity = ((fill / NSTAGE) & 1u) ^ 1u;
                auto open_stage = [&](uint64_t* full, uint32_t tx) {
                    if (lane == 0) asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(full)), "r"(tx) : "memory");
                    __syncwarp();
                };
                auto copy_group = [&](uint64_t* full) {
                    if (!OXI_IN_BOUNDS(c.row < p.batch && tok + nk <= c.slen && ps < (uint32_t)PAGES && id < p.map.num_blocks, status))
                        asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(full)), "r"(nk * Q8_ROW_BYTES) : "memory");
                    else
                        bulk_g2s_hint(dst, src, nk * Q8_ROW_BYTES, full, policy);
                };
                if (fill >= NSTAGE && !mbar_wait_bounded(&k_empty[slot], parity, abort_flag, wait_us)) {
                    ok = false;
                    break;
                }
                // test support: this CTA's stage goes missing
                if (fault.skip_plus1 && blockIdx.x == 0 && fill + 1u == fault.skip_plus1) continue;
                open_stage(&k_full[slot], bytes + (first ? Q_BYTES : 0));
                if (lane < NGROUP) {
                    if (live) copy_group(&k_full[slot]);
                } else if (first && lane == 2 * NGROUP) {
                    bulk_g2s(sbase + Q_OFF, reinterpret_cast<const char*>(p.q) + (size_t)c.row * Q_BYTES, Q_BYTES, &k_full[slot]);
                }
                if (lane < NGROUP) {
                    reinterpret_cast<uint16_t*>(sb + DESC_OFF + 16)[lane] = (uint16_t)vis;
                    sb[DESC_OFF + 24 + lane] = (unsigned char)ps;
                }
                if (lane == 0)
                    *reinterpret_cast<uint4*>(sb + DESC_OFF) =
                        make_uint4(c.row, c.range | (nchunks << 16), (nitem % NTABLE) | (first ? F_FIRST : 0u) | (last ? F_LAST : 0u), 0u);
                if (first) {
                    // the item's scales; the stage is full when they too have arrived
                    if ((uint32_t)lane < c.np && lane < PAGES) {
                        const uint32_t to = smem_u32(table + 32 * lane);
                        const size_t at = (size_t)c.id * p.map.scale_stride;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p.map.k_scales + at) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16u), "l"(p.map.v_scales + at) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(smem_u32(&k_full[slot])) : "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[slot]);
                if (fill >= NSTAGE && !mbar_wait_bounded(&v_empty[slot], parity, abort_flag, wait_us)) {
                    ok = false;
                    break;
                }
                open_stage(&v_full[slot], bytes);
                if (is_v && lane < 2 * NGROUP && live) copy_group(&v_full[slot]);
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[slot]);
            }
            cur = nxt;
            nxt = nxt2;
            c = n;
            n = m;
            nxt2 = nxt < total_items ? answer() : total_items;
            if (nxt2 < total_items) {
                ask();
                m = open_item(nxt2);
            }
            ++nitem;
        }
        if (ok) {
            const uint32_t slot = fill % NSTAGE;
            if (fill < NSTAGE || mbar_wait_bounded(&k_empty[slot], ((fill / NSTAGE) & 1u) ^ 1u, abort_flag, wait_us)) {
                if (lane == 0) {
                    *reinterpret_cast<uint4*>(smem + (size_t)slot * STAGE_BYTES + DESC_OFF) = make_uint4(0u, 0u, F_END, 0u);
                    mbar_arrive(&k_full[slot]);
                }
            } else {
                ok = false;
            }
        }
        if (!ok) {
            // give the copies already issued a bounded time to land before this CTA's shared memory is released
            if (lane == 0) atomicOr(status, DEV_WAIT_TIMEOUT);
            for (uint32_t k = fill > NSTAGE ? fill - NSTAGE : 0; k <= fill; ++k) {
                mbar_wait_drain(&k_full[k % NSTAGE], (k / NSTAGE) & 1u, wait_us);
                mbar_wait_drain(&v_full[k % NSTAGE], (k / NSTAGE) & 1u, wait_us);
            }
        }
        return;
    }

    // ============================= consumer warps =============================
    const int kvh = warp, g = lane >> 2, t4 = lane & 3;
    const uint64_t keep_policy = l2_policy_evict_last();
    uint32_t qb[8][2];       // Q^T fragments: column (head) g, the dims of k-step s in the K codes' order
    float o[8][4];           // O^T: tile d, rows g (dim 16d + 2g) and g + 8 (dim 16d + 2g + 1), columns (heads) 2 t4, 2 t4 + 1
    float m0 = -1.0e30f, m1 = -1.0e30f, l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; s++) qb[s][0] = qb[s][1] = 0u;

    for (uint32_t take = 0;; ++take) {
        const uint32_t slot = take % NSTAGE;
        if (!mbar_wait_bounded(&k_full[slot], (take / NSTAGE) & 1u, abort_flag, wait_us)) {
            if (lane == 0) atomicOr(status, DEV_WAIT_TIMEOUT);
            break;
        }
        unsigned char* sb = smem + (size_t)slot * STAGE_BYTES;
        const uint4 desc = *reinterpret_cast<const uint4*>(sb + DESC_OFF);
        if (desc.z & F_END) break;
        const uint2 vis2 = *reinterpret_cast<const uint2*>(sb + DESC_OFF + 16);
        const bool whole = (vis2.x & vis2.y) == 0xffffffffu;
        const uint32_t gg = g & 3u, gt = g >> 2;  // this thread's group, and its first token in it
        const uint32_t vis = reinterpret_cast<const uint16_t*>(sb + DESC_OFF + 16)[gg], ps = sb[DESC_OFF + 24 + gg];

        if (desc.z & F_FIRST) {
            const unsigned char* qrow = sb + Q_OFF + (kvh * 4 + (g & 3)) * (HD * 2);
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const uint2 d = *reinterpret_cast<const uint2*>(qrow + (16 * (t4 + 4 * (s >> 2)) + 4 * (s & 3)) * 2);
                qb[s][0] = g < 4 ? d.x : 0u;
                qb[s][1] = g < 4 ? d.y : 0u;
            }
#pragma unroll
            for (int d = 0; d < 8; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
            m0 = m1 = -1.0e30f;
            l0 = l1 = 0.0f;
        }
        const float* table = reinterpret_cast<const float*>(tables + (desc.z & 0xffffu) * TABLE_BYTES) + ps * 8 + kvh;
        float ks = table[0], vs = table[4];
        if (!whole) {
            if (vis == 0u) ks = vs = 0.0f;  // no group: its scales are not in the table
        }
        const float xs = ks * X_SCALE;
        const float lv = fmaxf(__log2f(vs), Q8_V_SCALE_MIN_LOG2), ivs = exp2f(-lv);

        // ---- S^T: tile i holds tokens 4i and 4i + 1 of the 4 groups in rows 0-7 and tokens 4i + 2 and 4i + 3 in rows 8-15
        // (the four tiles side by side: their accumulations are independent)
        float s[4][4];
        const unsigned char* krow = sb + gg * KPITCH + gt * Q8_ROW_BYTES + kvh * HD + t4 * 16;
#pragma unroll
        for (int i = 0; i < 4; i++) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            uint4 kc[8];
#pragma unroll
            for (int i = 0; i < 8; i++) kc[i] = *reinterpret_cast<const uint4*>(krow + 2 * i * Q8_ROW_BYTES + hf * 64);
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t aw = j == 0 ? kc[2 * i].x : j == 1 ? kc[2 * i].y : j == 2 ? kc[2 * i].z : kc[2 * i].w;
                    const uint32_t bw = j == 0 ? kc[2 * i + 1].x : j == 1 ? kc[2 * i + 1].y : j == 2 ? kc[2 * i + 1].z : kc[2 * i + 1].w;
                    uint32_t a0, a1, a2, a3;
                    codes_to_f16<kFmt>(aw, a0, a2);
                    codes_to_f16<kFmt>(bw, a1, a3);
                    mma_free(s[i], a0, a1, a2, a3, qb[4 * hf + j][0], qb[4 * hf + j][1]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_empty[slot]);
        if (!mbar_wait_bounded(&v_full[slot], (take / NSTAGE) & 1u, abort_flag, wait_us)) {
            if (lane == 0) atomicOr(status, DEV_WAIT_TIMEOUT);
            break;
        }
        if (!whole) {
            // codes that are not visible may be anything (an e4m3 NaN times the weight 0 would be a NaN)
            for (uint32_t i = lane; i < KS * 8u; i += 32) {
                const uint32_t key = i >> 3;
                if (!(((key < 32u ? vis2.x : vis2.y) >> (key & 31u)) & 1u))
                    *reinterpret_cast<uint4*>(sb + V_OFF + (key / GK) * VPITCH + (key % GK) * Q8_ROW_BYTES + kvh * HD + (i & 7u) * 16u) =
                        make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
        }
        // the first V codes, while the scores settle: k-step i of PV has the keys of tile i in the same order
        const uint32_t vaddr = smem_u32(sb) + V_OFF + (lane & 3) * VPITCH + (((lane >> 2) & 1) + 2 * (lane >> 3)) * Q8_ROW_BYTES + kvh * HD;
        uint32_t r[4][4];
        auto load_v = [&](int i2, int d4) {
#pragma unroll
            for (int d = 0; d < 4; d++) ldmatrix_x4_trans(vaddr + i2 * 8 * Q8_ROW_BYTES + (d4 + d) * 16, r[d][0], r[d][1], r[d][2], r[d][3]);
        };
        load_v(0, 0);
        // ---- exponents; the maxima of the two heads only where one of them has to be raised
        float n0 = -INFINITY, n1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float e = fmaf(s[i][j], xs, lv);
                s[i][j] = (whole || ((vis >> (4 * i + 2 * (j >> 1) + gt)) & 1u)) ? e : -INFINITY;
            }
            n0 = fmaxf(n0, fmaxf(s[i][0], s[i][2]));
            n1 = fmaxf(n1, fmaxf(s[i][1], s[i][3]));
        }
        if (__any_sync(0xffffffffu, n0 > m0 + RAISE || n1 > m1 + RAISE)) {
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, off));
                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, off));
            }
            n0 = fmaxf(n0, m0);
            n1 = fmaxf(n1, m1);
            const float c0 = ex2_approx_ftz(m0 - n0), c1 = ex2_approx_ftz(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= c0;
            l1 *= c1;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                o[d][0] *= c0;
                o[d][1] *= c1;
                o[d][2] *= c0;
                o[d][3] *= c1;
            }
        }
        // ---- weights, and their transposition into the B operand
        float p0 = 0.0f, p1 = 0.0f;
        uint32_t pb[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float w0 = ex2_approx_ftz(s[i][0] - m0), w1 = ex2_approx_ftz(s[i][1] - m1);
            const float w2 = ex2_approx_ftz(s[i][2] - m0), w3 = ex2_approx_ftz(s[i][3] - m1);
            p0 += w0 + w2;
            p1 += w1 + w3;
            pb[i][0] = transpose_8x8(pack_h2(w0, w1));
            pb[i][1] = transpose_8x8(pack_h2(w2, w3));
        }
        l0 = fmaf(p0, ivs, l0);
        l1 = fmaf(p1, ivs, l1);
        // ---- O^T += V^T P^T
#pragma unroll
        for (int i2 = 0; i2 < 2; i2++) {
#pragma unroll
            for (int d4 = 0; d4 < 8; d4 += 4) {
                if (i2 + d4 > 0) load_v(i2, d4);
#pragma unroll
                for (int j = 0; j < 2; j++) {
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        uint32_t a0, a1, a2, a3;
                        codes_to_f16<kFmt>(__byte_perm(r[d][2 * j], 0u, 0x3120), a0, a1);
                        codes_to_f16<kFmt>(__byte_perm(r[d][2 * j + 1], 0u, 0x3120), a2, a3);
                        mma_free(o[d4 + d], a0, a1, a2, a3, pb[2 * i2 + j][0], pb[2 * i2 + j][1]);
                    }
                }
            }
        }
        if (!whole) fence_proxy_async_smem();  // the zeros above, before the next copy into this stage
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[slot]);
        if (!(desc.z & F_LAST)) continue;

        // ---- the item is complete
        const uint32_t b = desc.x, rg = desc.y & 0xffffu, nchunks = desc.y >> 16;
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, off);
            l1 += __shfl_xor_sync(0xffffffffu, l1, off);
        }
        const uint32_t head = kvh * 4 + 2 * (t4 & 1);
        if (t4 >= 2) {  // columns 4-7 hold no heads
        } else if (nchunks == 1) {
            float f0 = rcp_approx_ftz(l0), f1 = rcp_approx_ftz(l1);
            if (p.gate) {
                f0 *= sigmoid_ref(h2f(p.gate[(size_t)b * NQ + head]));
                f1 *= sigmoid_ref(h2f(p.gate[(size_t)b * NQ + head + 1]));
            }
            uint16_t* out = p.ctx_out + ((size_t)b * NQ + head) * HD;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                *reinterpret_cast<uint32_t*>(out + 16 * d + 2 * g) = pack_h2(o[d][0] * f0, o[d][2] * f0);
                *reinterpret_cast<uint32_t*>(out + HD + 16 * d + 2 * g) = pack_h2(o[d][1] * f1, o[d][3] * f1);
            }
        } else if (OXI_IN_BOUNDS(b < p.batch && rg < p.ws.max_chunks && nchunks <= p.ws.max_chunks, status)) {
            const size_t pslot = ((size_t)b * p.ws.max_chunks + rg) * NQ + head;
            float* acc = p.ws.partial_acc + pslot * HD;
#pragma unroll
            for (int d = 0; d < 8; d++) {
                st_global_f2_hint(acc + 16 * d + 2 * g, o[d][0], o[d][2], keep_policy);
                st_global_f2_hint(acc + HD + 16 * d + 2 * g, o[d][1], o[d][3], keep_policy);
            }
            if (g == 0) {
                st_global_f2_hint(p.ws.partial_stats + pslot * 2, m0, l0, keep_policy);
                st_global_f2_hint(p.ws.partial_stats + (pslot + 1) * 2, m1, l1, keep_policy);
            }
        }
        __syncwarp();
    }
}

cudaError_t decode_attn_q8_init() {
    cudaError_t e = cudaFuncSetAttribute(decode_attn_q8_kernel<Q8_INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dq::SMEM_BYTES);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(decode_attn_q8_kernel<Q8_E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dq::SMEM_BYTES);
    return e;
}

cudaError_t launch_decode_attn_q8(cudaStream_t stream, const DecodeWorkspace& ws, void* ctx_out, const void* q, const void* gate,
                                  const Q8Map& map, uint32_t format, const uint32_t* seq_lens, uint32_t batch, uint32_t window,
                                  uint32_t sinks) {
    DecodeQ8Params p;
    p.ctx_out = (uint16_t*)ctx_out;
    p.q = (const uint16_t*)q;
    p.gate = (const uint16_t*)gate;
    p.map = map;
    p.seq_lens = seq_lens;
    p.ws = ws;
    p.batch = batch;
    p.window = window;
    p.sinks = sinks;
    p.direct = view_is_one_range(window, sinks, dq::CHUNK_G, dq::GK) || ws.max_seq_len <= (uint32_t)dq::CHUNK;  // nothing to merge
    const cudaError_t e = launch_pdl(format == Q8_INT8 ? decode_attn_q8_kernel<Q8_INT8> : decode_attn_q8_kernel<Q8_E4M3>,
                                     dim3(ws.num_sms), dim3(dq::THREADS), dq::SMEM_BYTES, stream, p);
    if (e != cudaSuccess || p.direct) return e;
    return launch_decode_merge_q8(stream, ws, ctx_out, gate, map, seq_lens, batch, window, sinks);
}

}  // namespace oxi
