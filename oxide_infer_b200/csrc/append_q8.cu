// RMSNorm + RoPE of q and k and the quantising append of k and v to the 8-bit paged cache, one launch for
// decode rows and for prefill waves.
//
//   y = x / sqrt(mean(x^2) + eps) * w,   z[d] = y[d] cos[d] - y[d+64] sin[d],   z[d+64] = y[d+64] cos[d+64] + y[d] sin[d+64]
//   q_out = f16(z);   k code = round(z / s_k),   v code = round(v / s_v)
//
// with s the scale of the token's (block, KV head).  A scale belongs to a whole block, so the rows of a run that
// fall into one block (a segment) need their largest magnitude first; then the block's new scale, requantised codes
// of the slots before the segment if the scale grew, and the segment's codes.  Nothing waits on another CTA.
//
// Two kernels, by what the caller passes: without row_seq every row is a segment of its own (append_q8_step_kernel),
// with it rows may form runs (append_q8_wave_kernel).
//
// Dims are spread over lanes so that both members of every rotation pair are in one lane and all accesses of a warp
// are contiguous.
#include "kernels.h"
#include "q8.cuh"

namespace oxi {

namespace aq {
constexpr float F16_MAX = 65504.0f;
constexpr int COMBOS = 2 * NKV;                    // K or V of a KV head
constexpr int STEP_THREADS = (NQ + COMBOS) * 32;   // a warp for each head of the row
constexpr int WAVE_WARPS = 16, WAVE_THREADS = WAVE_WARPS * 32;
constexpr int KV_PAIRS = NKV;                      // pairs of K or V heads of a row: K 0-1, K 2-3, V 0-1, V 2-3
constexpr int Q_PARTS = 2, Q_PAIRS = NQ / 2 / Q_PARTS;  // CTAs for a window's query heads, pairs of heads of a warp there
}  // namespace aq

struct AppendQ8Params {
    uint16_t* q_out;
    const uint16_t* q_in;
    const uint16_t* k_in;
    const uint16_t* v_in;
    const uint16_t* q_norm_w;
    const uint16_t* k_norm_w;
    const uint16_t* cos_t;
    const uint16_t* sin_t;
    const uint32_t* pos_ids;
    const uint32_t* row_seq;  // may be null
    Q8Map map;
    uint32_t rows;
    uint32_t max_seq_len;
    float eps;
    uint32_t* status;
};

// dims 2l, 2l+1, 64+2l, 65+2l of 128 consecutive f16
__device__ __forceinline__ void load_pairs(const uint16_t* p, int lane, float (&x)[4]) {
    const __half2 a = reinterpret_cast<const __half2*>(p)[lane], b = reinterpret_cast<const __half2*>(p)[32 + lane];
    x[0] = __low2float(a);
    x[1] = __high2float(a);
    x[2] = __low2float(b);
    x[3] = __high2float(b);
}

__device__ __forceinline__ void norm_rope_pairs(float (&x)[4], const float (&w)[4], const float (&c)[4], const float (&s)[4], float eps) {
    float sum = fmaf(x[0], x[0], fmaf(x[1], x[1], fmaf(x[2], x[2], x[3] * x[3])));
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float r = rsqrtf(fmaf(sum, 1.0f / HD, eps));
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = x[i] * r * w[i];
    x[0] = fmaf(y[0], c[0], -y[2] * s[0]);
    x[1] = fmaf(y[1], c[1], -y[3] * s[1]);
    x[2] = fmaf(y[2], c[2], y[0] * s[2]);
    x[3] = fmaf(y[3], c[3], y[1] * s[3]);
}

// Infinite and NaN values and values beyond f16 are stored as +-65504 and 0; returns whether there were any.
__device__ __forceinline__ bool make_finite(float (&x)[4]) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (!(fabsf(x[j]) <= aq::F16_MAX)) {
            odd = true;
            x[j] = x[j] != x[j] ? 0.0f : copysignf(aq::F16_MAX, x[j]);
        }
    }
    return odd;
}

__device__ __forceinline__ float abs_max(const float (&x)[4]) {
    return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}

__device__ __forceinline__ void store_q(uint16_t* head, int lane, const float (&x)[4]) {
    reinterpret_cast<uint32_t*>(head)[lane] = pack_h2(x[0], x[1]);
    reinterpret_cast<uint32_t*>(head)[32 + lane] = pack_h2(x[2], x[3]);
}

template <uint32_t kFmt>
__device__ __forceinline__ void store_codes(unsigned char* at, int lane, const float (&x)[4], float inv) {
    reinterpret_cast<uint16_t*>(at)[lane] = (uint16_t)q8_codes2<kFmt>(x[0], x[1], inv);
    reinterpret_cast<uint16_t*>(at)[32 + lane] = (uint16_t)q8_codes2<kFmt>(x[2], x[3], inv);
}

// Row r is a token of table row r.  grid = rows, a warp for each query head, K head and V head; all of them share the
// slots to requantise where a scale grew.  128 rows: 1.8 us if none grows; if all do in the last slot of a block, int8 6.2 us in
// blocks of 16 and 39 in blocks of 256 (e4m3 5.8 and 34; 67 MB, 10 us of memory time).  In use a head's scale grows with a
// probability of about 1 / (slot + 1) (int8) or less (e4m3, whose scales are powers of two): on average over the tokens of a block
// with normally distributed values 3.0 us a step in blocks of 16 and 64 and 4.4 to 4.9 in blocks of 256, e4m3 2.4 to 2.8.
template <uint32_t kFmt>
__global__ void __launch_bounds__(aq::STEP_THREADS)
append_q8_step_kernel(const AppendQ8Params p) {
    using namespace aq;
    __shared__ float s_ratio[COMBOS];  // old scale / new scale of a head whose scale grew
    __shared__ uint32_t s_grown;
    const uint32_t r = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    if (threadIdx.x == 0) s_grown = 0u;
    __syncthreads();
    // the step's tables, norm weights and rotary rows are not written by any kernel: read while the preceding
    // kernel is still draining
    const uint32_t lbs = p.map.lbs, pos = p.pos_ids[r], blk = pos >> lbs, slot = pos & ((1u << lbs) - 1u);
    if (pos >= p.max_seq_len || blk >= p.map.max_blocks) {
        if (threadIdx.x == 0) atomicOr(p.status, DEV_BAD_SEQ_LEN);
        pdl_wait();
        return;
    }
    const int combo = warp - NQ;  // >= 0: K or V head
    const bool is_v = combo >= NKV;
    const uint32_t id = p.map.block_tables[(size_t)r * p.map.max_blocks + blk];
    const bool placed = id < p.map.num_blocks;
    auto head_codes = [&](int c) {
        return (c >= NKV ? p.map.v_pool : p.map.k_pool) + (size_t)id * p.map.block_stride + (c & (NKV - 1)) * HD;
    };
    float wv[4], cv[4], sv[4], x[4];
    if (!is_v) {
        load_pairs(combo < 0 ? p.q_norm_w : p.k_norm_w, lane, wv);
        load_pairs(p.cos_t + (size_t)pos * HD, lane, cv);
        load_pairs(p.sin_t + (size_t)pos * HD, lane, sv);
    }
    pdl_wait();  // q, k, v come from the preceding kernel; the cache may still be read by it
    if (combo < 0) {
        const size_t at = ((size_t)r * NQ + warp) * HD;
        load_pairs(p.q_in + at, lane, x);
        norm_rope_pairs(x, wv, cv, sv, p.eps);
        store_q(p.q_out + at, lane, x);
    } else if (!placed) {
        if (combo == 0 && lane == 0) atomicOr(p.status, DEV_BAD_BLOCK);
    } else {
        const int kvh = combo & (NKV - 1);
        float* scale_at = (is_v ? p.map.v_scales : p.map.k_scales) + (size_t)id * p.map.scale_stride + kvh;
        const float old_scale = slot != 0u ? __ldcg(scale_at) : 0.0f;
        load_pairs((is_v ? p.v_in : p.k_in) + ((size_t)r * NKV + kvh) * HD, lane, x);
        if (!is_v) norm_rope_pairs(x, wv, cv, sv, p.eps);
        if (__any_sync(0xffffffffu, make_finite(x)) && lane == 0) atomicOr(p.status, DEV_NONFINITE);
        const float scale = fmaxf(q8_scale<kFmt>(warp_max(abs_max(x))), old_scale);
        // bounds build: the token's slot lies in a block of the pool
        if (OXI_IN_BOUNDS(id < p.map.num_blocks && slot >> lbs == 0u, p.status)) store_codes<kFmt>(head_codes(combo) + (size_t)slot * Q8_ROW_BYTES, lane, x, q8_inverse<kFmt>(scale));
        if (lane == 0) {
            *scale_at = scale;
            if (slot != 0u && scale > old_scale) {
                s_ratio[combo] = __fdiv_rn(old_scale, scale);
                atomicOr(&s_grown, 1u << combo);
            }
        }
    }
    __syncthreads();
    // a unit is one slot's 128 codes of a head whose scale grew: four in flight per warp
    const uint32_t grown = s_grown, units = (uint32_t)__popc(grown) * slot;
    for (uint32_t u0 = warp; u0 < units; u0 += 4u * (NQ + COMBOS)) {
        uint32_t* at[4];
        uint32_t w[4];
        float ratio[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            const uint32_t u = min(u0 + k * (NQ + COMBOS), units - 1u), nth = u / slot;
            uint32_t m = grown;
            for (uint32_t i = 0; i < nth; i++) m &= m - 1u;
            const int c = __ffs((int)m) - 1;
            ratio[k] = s_ratio[c];
            at[k] = reinterpret_cast<uint32_t*>(head_codes(c) + (size_t)(u - nth * slot) * Q8_ROW_BYTES) + lane;
            w[k] = __ldcg(at[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            const uint32_t u = u0 + k * (NQ + COMBOS);
            // bounds build: the slot is one before the token's of a head whose scale grew, the block one of the pool
            if (u < units && OXI_IN_BOUNDS(u / slot < (uint32_t)__popc(grown) && slot >> lbs == 0u && id < p.map.num_blocks, p.status))
                *at[k] = q8_moved<kFmt>(w[k], ratio[k]);
        }
    }
}

// ---- the wave kernel's unit is a PAIR of heads of one row in a warp: lanes 0-15 hold the first, lanes 16-31 the second,
// lane j (mod 16) dims 4j .. 4j+3 and 64+4j .. 64+4j+3: eight-byte loads, and one reduction serves two heads.
__device__ __forceinline__ void load_dims(const uint16_t* head, int j, float (&x)[8]) {
    const uint2 a = reinterpret_cast<const uint2*>(head)[j], b = reinterpret_cast<const uint2*>(head)[16 + j];
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
// the same 8 dims of a norm weight, cos or sin row, kept as f16 pairs (registers)
struct Dims {
    uint32_t w[4];
    __device__ __forceinline__ float operator[](int i) const {
        const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
        return i & 1 ? __high2float(h) : __low2float(h);
    }
};
__device__ __forceinline__ Dims dims_of(const uint16_t* head, int j) {
    const uint2 a = reinterpret_cast<const uint2*>(head)[j], b = reinterpret_cast<const uint2*>(head)[16 + j];
    return Dims{{a.x, a.y, b.x, b.y}};
}
__device__ __forceinline__ void norm_rope_dims(float (&x)[8], const Dims& w, const Dims& c, const Dims& s, float eps) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    const float r = rsqrtf(fmaf(sum, 1.0f / HD, eps));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * r * w[i];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float lo = x[i], hi = x[4 + i];
        x[i] = fmaf(lo, c[i], -hi * s[i]);
        x[4 + i] = fmaf(hi, c[4 + i], lo * s[4 + i]);
    }
}
// largest magnitude of the lane's head; infinite, NaN and too large values are replaced as in make_finite
__device__ __forceinline__ float head_max(float (&x)[8], bool& odd) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        bad |= !(fabsf(x[i]) <= aq::F16_MAX);
        m = fmaxf(m, fabsf(x[i]));
    }
    if (bad) {
        odd = true;
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (!(fabsf(x[i]) <= aq::F16_MAX)) x[i] = x[i] != x[i] ? 0.0f : copysignf(aq::F16_MAX, x[i]);
            m = fmaxf(m, fabsf(x[i]));
        }
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    return m;
}
template <uint32_t kFmt>
__device__ __forceinline__ void store_dims(unsigned char* head, int j, const float (&x)[8], float inv) {
    reinterpret_cast<uint32_t*>(head)[j] = q8_codes2<kFmt>(x[0], x[1], inv) | (q8_codes2<kFmt>(x[2], x[3], inv) << 16);
    reinterpret_cast<uint32_t*>(head)[16 + j] = q8_codes2<kFmt>(x[4], x[5], inv) | (q8_codes2<kFmt>(x[6], x[7], inv) << 16);
}

// Row r is a token of table row row_seq[r].  grid = (windows of 16 rows, kSplit + Q_PARTS), warp w has row w of the window.
// CTAs with y >= kSplit do query heads, with nothing to agree on; CTA y < kSplit takes one of kSplit groups of K and V heads
// for the segments that BEGIN in its window, to their end: rows behind the window (its last segment may go on for up to 255
// rows) are read twice, once for the scale and once for the codes.  Rows at the window's start that go on with a segment
// of the window before are left to that CTA.
template <uint32_t kFmt, int kSplit>
__global__ void __launch_bounds__(aq::WAVE_THREADS, 2)
append_q8_wave_kernel(const AppendQ8Params p) {
    using namespace aq;
    constexpr int ROWS = WAVE_WARPS;             // a warp for each row of the window
    constexpr int NP = KV_PAIRS / kSplit;        // K / V pairs of a warp
    // per row of the window; a segment is named by its first row
    __shared__ uint32_t s_pos[ROWS], s_seq[ROWS], s_id[ROWS], s_end[ROWS], s_bad[ROWS];
    __shared__ int s_lead[ROWS];  // the row's segment, -1: not of this CTA
    __shared__ uint32_t s_list[ROWS];  // the segments in order
    // slots whose codes move to a larger scale ("units"), by (segment, head): s_units[i] .. s_units[i + 1] are those of
    // (i / COMBOS, i % COMBOS)
    __shared__ uint32_t s_units[ROWS * COMBOS + 1];
    static_assert(ROWS * COMBOS == 128, "the units are summed up by four warps");
    __shared__ uint32_t s_part[4];
    __shared__ float s_amax[ROWS][COMBOS], s_old[ROWS][COMBOS], s_scale[ROWS][COMBOS], s_tailmax[ROWS][COMBOS];
    __shared__ uint32_t s_leaders, s_tail;
    const uint32_t row0 = blockIdx.x * ROWS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = lane >> 4, j = lane & 15;
    const int w = warp;                          // this warp's row of the window
    const int pair0 = (int)blockIdx.y * NP;      // and its first K / V pair
    const uint32_t lbs = p.map.lbs, bs = 1u << lbs;
    pdl_launch_dependents();
    // this warp's row, read by every warp itself: its rotary values are then on their way before the window is sorted out
    const uint32_t my_pos = row0 + w < p.rows ? p.pos_ids[row0 + w] : 0xffffffffu;
    const uint32_t my_seq = row0 + w < p.rows ? p.row_seq[row0 + w] : 0xffffffffu;
    const bool there = my_pos < p.max_seq_len && (my_pos >> lbs) < p.map.max_blocks && my_seq < p.map.table_rows;  // a row that is skipped is not read either
    const uint32_t pos = there ? my_pos : 0u;
    const Dims cv = dims_of(p.cos_t + (size_t)pos * HD, j), sv = dims_of(p.sin_t + (size_t)pos * HD, j);
    const size_t row = there ? row0 + w : 0u;
    if (blockIdx.y >= kSplit) {
        const Dims qw = dims_of(p.q_norm_w, j);
        pdl_wait();  // q comes from the preceding kernel
        if (!there) return;
        const size_t at = (row * NQ + 2 * Q_PAIRS * (blockIdx.y - kSplit) + half) * HD;
        Dims y[Q_PAIRS];
#pragma unroll
        for (int k = 0; k < Q_PAIRS; k++) y[k] = dims_of(p.q_in + at + 2 * k * HD, j);
#pragma unroll
        for (int k = 0; k < Q_PAIRS; k++) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = y[k][i];
            norm_rope_dims(v, qw, cv, sv, p.eps);
            uint16_t* out = p.q_out + at + 2 * k * HD;
            reinterpret_cast<uint2*>(out)[j] = make_uint2(pack_h2(v[0], v[1]), pack_h2(v[2], v[3]));
            reinterpret_cast<uint2*>(out)[16 + j] = make_uint2(pack_h2(v[4], v[5]), pack_h2(v[6], v[7]));
        }
        return;
    }
    if (tid == 0) s_tail = 256u;
    uint32_t block_id = 0;  // warp 0: the block of the segment that begins at row `lane`
    if (warp == 0) {
        const uint32_t r = row0 + (uint32_t)lane;
        uint32_t pos = 0, seq = 0, ppos = 0, pseq = 0;
        const bool there = lane < ROWS && r < p.rows;
        if (there) {
            pos = p.pos_ids[r];
            seq = p.row_seq[r];
            if (r > 0u) {
                ppos = p.pos_ids[r - 1u];
                pseq = p.row_seq[r - 1u];
            }
        }
        const bool valid = there && pos < p.max_seq_len && (pos >> lbs) < p.map.max_blocks && seq < p.map.table_rows;
        if (there && !valid && blockIdx.y == 0) atomicOr(p.status, DEV_BAD_SEQ_LEN);
        const bool leader = valid && ((pos & (bs - 1u)) == 0u || r == 0u || pseq != seq || ppos + 1u != pos);
        const uint32_t leaders = __ballot_sync(0xffffffffu, leader), valids = __ballot_sync(0xffffffffu, valid);
        if (lane < ROWS) {
            // a valid row that is no leader goes on with the row before; the row after one that is not valid is a leader
            const uint32_t upto = leaders & (0xffffffffu >> (31 - lane));
            s_lead[lane] = valid && upto ? 31 - __clz(upto) : -1;
            s_pos[lane] = valid ? pos : 0xffffffffu;
            s_seq[lane] = seq;
            // where the segment that begins here ends inside the window: the next leader or row that is not valid
            const uint32_t stop = (leaders | ~valids) & ~(0xffffffffu >> (31 - lane));
            s_end[lane] = min((uint32_t)ROWS, stop ? (uint32_t)__ffs((int)stop) - 1u : 32u);
            if (leader) block_id = p.map.block_tables[(size_t)seq * p.map.max_blocks + (pos >> lbs)];
            s_bad[lane] = 0u;
            if (leader) s_list[__popc(leaders & ((1u << lane) - 1u))] = lane;
        }
        if (lane == 0) s_leaders = leaders;
    }
    if (tid < ROWS * COMBOS) {
        s_amax[tid / COMBOS][tid % COMBOS] = 0.0f;
        s_tailmax[tid / COMBOS][tid % COMBOS] = 0.0f;
    }
    const Dims kw = dims_of(p.k_norm_w, j);
    __syncthreads();
    const uint32_t leaders = s_leaders;
    const int last = s_lead[ROWS - 1];
    if (tid < 256) {
        // rows behind the window that go on with its last row's segment: the first that does not ends the tail
        const uint32_t i = 1u + (uint32_t)tid, r = row0 + ROWS - 1u + i, lp = s_pos[ROWS - 1];
        const bool same = last >= 0 && (lp & (bs - 1u)) + i < bs && r < p.rows && p.row_seq[r] == s_seq[ROWS - 1] &&
                          p.pos_ids[r] == lp + i && lp + i < p.max_seq_len;
        if (!same) atomicMin(&s_tail, i - 1u);
    }
    __syncthreads();
    const uint32_t tail = s_tail;
    // another run of this call in a segment's block would race with it: both are refused (a thread for each segment and
    // four rows of the call)
    const uint32_t quads = (p.rows + 3u) / 4u, nsegs = (uint32_t)__popc(leaders), looks = nsegs * quads;
    const bool aligned = (((uintptr_t)p.row_seq) & 15u) == 0u;
    for (uint32_t i = tid; i < looks; i += WAVE_THREADS) {
        const uint32_t rank = nsegs == 1u ? 0u : i / quads, r0 = (i - rank * quads) * 4u, li = s_list[rank], seq = s_seq[li];
        uint4 q = make_uint4(~seq, ~seq, ~seq, ~seq);
        if (aligned && r0 + 4u <= p.rows) {
            q = *reinterpret_cast<const uint4*>(p.row_seq + r0);
        } else {
            q.x = p.row_seq[r0];
            if (r0 + 1u < p.rows) q.y = p.row_seq[r0 + 1u];
            if (r0 + 2u < p.rows) q.z = p.row_seq[r0 + 2u];
            if (r0 + 3u < p.rows) q.w = p.row_seq[r0 + 3u];
        }
        auto look = [&](uint32_t r, uint32_t s) {
            if (s != seq || (r >= row0 + li && r < row0 + s_end[li] + ((int)li == last ? tail : 0u))) return;
            const uint32_t at = p.pos_ids[r];
            if ((at >> lbs) == (s_pos[li] >> lbs) && at < p.max_seq_len) s_bad[li] = 1u;
        };
        look(r0, q.x);
        look(r0 + 1u, q.y);
        look(r0 + 2u, q.z);
        look(r0 + 3u, q.w);
    }
    if (warp == 0 && lane < ROWS) s_id[lane] = block_id;
    __syncthreads();
    pdl_wait();  // k and v come from the preceding kernel; the cache may still be read by it
    // heads of pair i: K (i < 2) or V, heads 2 (i mod 2) and + 1; combination (K 0-3, V 0-3) of this lane's head
    auto combo_of = [&](int i) { return 2 * i + half; };
    auto kv_head = [&](int i, size_t row) {
        return (i < KV_PAIRS / 2 ? p.k_in : p.v_in) + (row * NKV + 2 * (i % (KV_PAIRS / 2)) + half) * HD;
    };
    float x[NP][8];
#pragma unroll
    for (int k = 0; k < NP; k++) load_dims(kv_head(pair0 + k, row), j, x[k]);
    if (tid < ROWS * COMBOS) {  // a segment that begins behind slot 0 starts from the block's scale
        const int li = tid / COMBOS, c = tid % COMBOS;
        const bool read = ((leaders >> li) & 1u) && s_id[li] < p.map.num_blocks && (s_pos[li] & (bs - 1u)) != 0u;
        s_old[li][c] = read ? __ldcg((c < NKV ? p.map.k_scales : p.map.v_scales) + (size_t)s_id[li] * p.map.scale_stride + (c & (NKV - 1))) : 0.0f;
    }
    bool odd = false;
#pragma unroll
    for (int k = 0; k < NP; k++) {
        if (pair0 + k < KV_PAIRS / 2) norm_rope_dims(x[k], kw, cv, sv, p.eps);
        bool o = false;
        const float a = head_max(x[k], o);
        if (there && s_lead[w] >= 0) {
            odd |= o;
            if (j == 0) s_amax[w][combo_of(pair0 + k)] = a;
        }
    }
    // rows behind the window: row t of the tail by warp t mod 16
    auto tail_row = [&](uint32_t t, int i, float (&v)[8]) {
        load_dims(kv_head(i, row0 + ROWS + t), j, v);
        if (i < KV_PAIRS / 2) {
            const size_t at = s_pos[ROWS - 1] + 1u + t;
            norm_rope_dims(v, kw, dims_of(p.cos_t + at * HD, j), dims_of(p.sin_t + at * HD, j), p.eps);
        }
        return head_max(v, odd);
    };
#pragma unroll
    for (int k = 0; k < NP; k++) {
        float m = 0.0f;
#pragma unroll 2
        for (uint32_t t = w; t < tail; t += ROWS) {
            float v[8];
            m = fmaxf(m, tail_row(t, pair0 + k, v));
        }
        if (j == 0) s_tailmax[w][combo_of(pair0 + k)] = m;
    }
    if (__any_sync(0xffffffffu, odd) && lane == 0) atomicOr(p.status, DEV_NONFINITE);
    __syncthreads();
    uint32_t grown = 0;  // tid < ROWS * COMBOS: units of (segment, head)
    if (tid < ROWS * COMBOS && ((leaders >> (tid / COMBOS)) & 1u)) {
        const int li = tid / COMBOS, c = tid % COMBOS;
        float amax = 0.0f;
        for (uint32_t i = li; i < s_end[li]; i++) amax = fmaxf(amax, s_amax[i][c]);
        if (li == last)
            for (int i = 0; i < ROWS; i++) amax = fmaxf(amax, s_tailmax[i][c]);
        const float scale = fmaxf(q8_scale<kFmt>(amax), s_old[li][c]);
        s_scale[li][c] = scale;
        const bool no_block = s_id[li] >= p.map.num_blocks;
        if (no_block || s_bad[li]) {
            if (c == 0 && blockIdx.y == 0) atomicOr(p.status, no_block ? DEV_BAD_BLOCK : DEV_BLOCK_CONFLICT);
        } else if (c / (COMBOS / kSplit) == (int)blockIdx.y) {
            ((c < NKV ? p.map.k_scales : p.map.v_scales) + (size_t)s_id[li] * p.map.scale_stride)[c & (NKV - 1)] = scale;
            if (scale > s_old[li][c]) grown = s_pos[li] & (bs - 1u);
        }
    }
    if (tid < ROWS * COMBOS) {
        uint32_t sum = grown;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += t;
        }
        s_units[tid + 1] = sum;  // within the warp; the warps before are added below
        if (lane == 31) s_part[warp] = sum;
        if (tid == 0) s_units[0] = 0u;
    }
    __syncthreads();
    if (tid < ROWS * COMBOS && warp > 0) {
        uint32_t before = s_part[0];
        for (int i = 1; i < warp; i++) before += s_part[i];
        s_units[tid + 1] += before;
    }
    __syncthreads();
    auto usable = [&](int li) { return s_id[li] < p.map.num_blocks && s_bad[li] == 0u; };
    auto head_codes = [&](int li, int c) {  // this head's codes in the segment's block
        return (c < NKV ? p.map.k_pool : p.map.v_pool) + (size_t)s_id[li] * p.map.block_stride + (c & (NKV - 1)) * HD;
    };
    // four units in flight per warp
    const uint32_t units = s_units[ROWS * COMBOS];
    uint32_t i = 0;
    for (uint32_t u0 = w; u0 < units; u0 += 4u * ROWS) {
        uint32_t* at[4];
        uint32_t v[4];
        float ratio[4];
        bool inside[4];  // bounds build: the slot lies before its segment, and the segment's block in the pool
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            const uint32_t u = min(u0 + k * ROWS, units - 1u);
            while (s_units[i + 1] <= u) i++;
            const int sl = i / COMBOS, c = i % COMBOS;
            ratio[k] = __fdiv_rn(s_old[sl][c], s_scale[sl][c]);
            at[k] = reinterpret_cast<uint32_t*>(head_codes(sl, c) + (size_t)(u - s_units[i]) * Q8_ROW_BYTES) + lane;
            inside[k] = OXI_IN_BOUNDS(i < (uint32_t)(ROWS * COMBOS) && u - s_units[i] < (s_pos[sl] & (bs - 1u)) && s_id[sl] < p.map.num_blocks, p.status);
            if (inside[k]) v[k] = __ldcg(at[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            if (u0 + k * ROWS < units && inside[k]) *at[k] = q8_moved<kFmt>(v[k], ratio[k]);
    }
    const int li = there ? s_lead[w] : -1;
    if (li >= 0 && usable(li)) {
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int c = combo_of(pair0 + k);
            // bounds build: the row is the wave's, its block in the pool and its segment's
            if (OXI_IN_BOUNDS(row < p.rows && s_id[li] < p.map.num_blocks && pos >> lbs == s_pos[li] >> lbs, p.status))
                store_dims<kFmt>(head_codes(li, c) + (size_t)(pos & (bs - 1u)) * Q8_ROW_BYTES, j, x[k], q8_inverse<kFmt>(s_scale[li][c]));
        }
    }
    if (tail != 0u && usable(last)) {
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int c = combo_of(pair0 + k);
            const float inv = q8_inverse<kFmt>(s_scale[last][c]);
#pragma unroll 2
            for (uint32_t t = w; t < tail; t += ROWS) {
                float v[8];
                tail_row(t, pair0 + k, v);
                // bounds build: the row is the wave's and lies in the block of the window's last row
                if (OXI_IN_BOUNDS(row0 + ROWS + t < p.rows && s_id[last] < p.map.num_blocks &&
                                      (s_pos[ROWS - 1] + 1u + t) >> lbs == s_pos[last] >> lbs, p.status))
                    store_dims<kFmt>(head_codes(last, c) + (size_t)((s_pos[ROWS - 1] + 1u + t) & (bs - 1u)) * Q8_ROW_BYTES, j, v, inv);
            }
        }
    }
}

template <uint32_t kFmt, int kSplit>
static cudaError_t launch_wave(cudaStream_t stream, const AppendQ8Params& p) {
    return launch_pdl(append_q8_wave_kernel<kFmt, kSplit>, dim3((p.rows + aq::WAVE_WARPS - 1) / aq::WAVE_WARPS, kSplit + aq::Q_PARTS), dim3(aq::WAVE_THREADS), 0,
                      stream, p);
}

template <uint32_t kFmt>
static cudaError_t launch_fmt(cudaStream_t stream, const AppendQ8Params& p) {
    if (!p.row_seq) return launch_pdl(append_q8_step_kernel<kFmt>, dim3(p.rows), dim3(aq::STEP_THREADS), 0, stream, p);
    // How many CTAs share a window's K and V heads.  More of them give a long segment's rows more warps (rows behind the
    // window are serial work), fewer repeat a window's set-up less often; two CTAs fit an SM.  Measured, us, for 1 / 2 / 4
    // groups: 128 rows in one run, blocks of 16: 4.6 / 3.4 / 2.7, of 256: 27.9 / 19.1 / 10.9; 4,096 rows in runs of 128,
    // blocks of 16: 13.3 / 16.0 / 22.7, of 64: 23.2 / 18.2 / 22.0, of 256: 40.2 / 28.5 / 23.8 (between these points nothing was measured).
    if (p.rows <= 1184u || p.map.lbs > 6u) return launch_wave<kFmt, 4>(stream, p);
    return p.map.lbs == 6u ? launch_wave<kFmt, 2>(stream, p) : launch_wave<kFmt, 1>(stream, p);
}

cudaError_t launch_append_q8(cudaStream_t stream, void* q_out, const void* q_in, const void* k_in, const void* v_in,
                             const void* q_norm_w, const void* k_norm_w, const void* cos_t, const void* sin_t,
                             const uint32_t* pos_ids, const uint32_t* row_seq, const Q8Map& map, uint32_t format, uint32_t rows,
                             uint32_t max_seq_len, float eps, uint32_t* status) {
    AppendQ8Params p;
    p.q_out = (uint16_t*)q_out;
    p.q_in = (const uint16_t*)q_in;
    p.k_in = (const uint16_t*)k_in;
    p.v_in = (const uint16_t*)v_in;
    p.q_norm_w = (const uint16_t*)q_norm_w;
    p.k_norm_w = (const uint16_t*)k_norm_w;
    p.cos_t = (const uint16_t*)cos_t;
    p.sin_t = (const uint16_t*)sin_t;
    p.pos_ids = pos_ids;
    p.row_seq = row_seq;
    p.map = map;
    p.rows = rows;
    p.max_seq_len = max_seq_len;
    p.eps = eps;
    p.status = status;
    return format == Q8_INT8 ? launch_fmt<Q8_INT8>(stream, p) : launch_fmt<Q8_E4M3>(stream, p);
}

}  // namespace oxi
