// RMSNorm + RoPE of q and k and the quantising append of k and v to the 8-bit paged cache, one launch for
// decode rows and for prefill waves.
//
//   y = x / sqrt(mean(x^2) + eps) * w,   z[d] = y[d] cos[d] - y[d+64] sin[d],   z[d+64] = y[d+64] cos[d+64] + y[d] sin[d+64]
//   q_out = f16(z);   k code = round(z / s_k),   v code = round(v / s_v)
//
// with s the scale of the token's (block, KV head).  A scale belongs to a whole block, so the rows of a run that
// fall into one block are handled together by the CTA of the first of them (the segment's leader): largest
// magnitude over the segment, the block's new scale, requantised codes of the slots before the segment if the
// scale grew, then the segment's codes.  Nothing waits on another CTA: the leader reads the whole segment, the
// CTAs of the other rows only do their q.
//
// grid = rows, 16 warps: warp w does q head w; in a leader's CTA warp w then does every second row of the
// segment for (K or V, KV head) = w mod 8.  Lane l holds dims 2l, 2l+1, 64+2l, 65+2l, so that both members of
// every rotation pair sit in one lane.
#include "kernels.h"
#include "q8.cuh"

namespace oxi {

namespace aq {
constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int COMBOS = 2 * NKV;             // K or V of a KV head
constexpr int PARTS = WARPS / COMBOS;       // warps that share a combination's rows
constexpr int KEEP = 8;                     // rows a warp keeps in registers between the two passes
constexpr float F16_MAX = 65504.0f;
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

template <uint32_t kFmt>
__global__ void __launch_bounds__(aq::THREADS)
append_q8_kernel(const AppendQ8Params p) {
    using namespace aq;
    __shared__ uint32_t s_len, s_conflict;
    __shared__ float s_amax[PARTS][COMBOS];
    const uint32_t r = blockIdx.x;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    if (tid == 0) {
        s_len = 0xffffffffu;
        s_conflict = 0u;
    }
    // the step's tables, norm weights and rotary rows are not written by any kernel: read while the preceding
    // kernel is still draining
    const uint32_t lbs = p.map.lbs, bs = 1u << lbs;
    const uint32_t pos = p.pos_ids[r];
    const uint32_t seq = p.row_seq ? p.row_seq[r] : r;
    const uint32_t blk = pos >> lbs, slot0 = pos & (bs - 1u);
    if (pos >= p.max_seq_len || blk >= p.map.max_blocks) {
        if (tid == 0) atomicOr(p.status, DEV_BAD_SEQ_LEN);
        pdl_wait();
        return;
    }
    bool leader = slot0 == 0u || r == 0u || !p.row_seq;
    if (!leader) leader = p.row_seq[r - 1] != seq || p.pos_ids[r - 1] + 1u != pos;
    __syncthreads();
    uint32_t n = 1u, id = 0u;
    if (leader) {
        if (p.row_seq) {
            // length of the segment: rows that go on with the next position of the same sequence inside the block
            for (uint32_t i = 1u + tid; slot0 + i <= bs; i += THREADS) {
                const bool same = slot0 + i < bs && r + i < p.rows && p.row_seq[r + i] == seq && p.pos_ids[r + i] == pos + i &&
                                  pos + i < p.max_seq_len;
                if (!same) {
                    atomicMin(&s_len, i);
                    break;
                }
            }
            __syncthreads();
            n = s_len;
            // another run of this call in the same block would race with this one
            for (uint32_t j = tid; j < p.rows; j += THREADS)
                if ((j < r || j >= r + n) && p.row_seq[j] == seq && (p.pos_ids[j] >> lbs) == blk && p.pos_ids[j] < p.max_seq_len) s_conflict = 1u;
        }
        id = p.map.block_tables[(size_t)seq * p.map.max_blocks + blk];
    }
    float wv[4], cv[4], sv[4];
    load_pairs(p.q_norm_w, lane, wv);
    load_pairs(p.cos_t + (size_t)pos * HD, lane, cv);
    load_pairs(p.sin_t + (size_t)pos * HD, lane, sv);
    pdl_wait();  // q, k, v come from the preceding kernel; the cache may still be read by it
    {
        float x[4];
        const size_t at = ((size_t)r * NQ + warp) * HD;
        load_pairs(p.q_in + at, lane, x);
        norm_rope_pairs(x, wv, cv, sv, p.eps);
        reinterpret_cast<uint32_t*>(p.q_out + at)[lane] = pack_h2(x[0], x[1]);
        reinterpret_cast<uint32_t*>(p.q_out + at)[32 + lane] = pack_h2(x[2], x[3]);
    }
    if (!leader) return;
    __syncthreads();
    if (id >= p.map.num_blocks || s_conflict) {
        if (tid == 0) atomicOr(p.status, s_conflict ? DEV_BLOCK_CONFLICT : DEV_BAD_BLOCK);
        return;
    }
    const int combo = warp & (COMBOS - 1), part = warp / COMBOS, kvh = combo & (NKV - 1);
    const bool is_v = combo >= NKV;
    float* scale_at = (is_v ? p.map.v_scales : p.map.k_scales) + (size_t)id * p.map.scale_stride + kvh;
    const float old_scale = slot0 != 0u ? __ldcg(scale_at) : 0.0f;
    if (!is_v) load_pairs(p.k_norm_w, lane, wv);
    bool odd = false;  // some value is not a finite f16
    auto load_row = [&](uint32_t i, float (&x)[4]) {
        load_pairs((is_v ? p.v_in : p.k_in) + ((size_t)(r + i) * NKV + kvh) * HD, lane, x);
        if (!is_v) {
            load_pairs(p.cos_t + (size_t)(pos + i) * HD, lane, cv);
            load_pairs(p.sin_t + (size_t)(pos + i) * HD, lane, sv);
            norm_rope_pairs(x, wv, cv, sv, p.eps);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (!(fabsf(x[j]) <= F16_MAX)) {
                odd = true;
                x[j] = x[j] != x[j] ? 0.0f : copysignf(F16_MAX, x[j]);
            }
        }
    };
    float keep[KEEP][4], amax = 0.0f;
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const uint32_t i = part + k * PARTS;
        if (i < n) {
            load_row(i, keep[k]);
#pragma unroll
            for (int j = 0; j < 4; j++) amax = fmaxf(amax, fabsf(keep[k][j]));
        }
    }
    for (uint32_t i = part + KEEP * PARTS; i < n; i += PARTS) {
        float x[4];
        load_row(i, x);
#pragma unroll
        for (int j = 0; j < 4; j++) amax = fmaxf(amax, fabsf(x[j]));
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (lane == 0) s_amax[part][combo] = amax;
    if (__any_sync(0xffffffffu, odd) && lane == 0) atomicOr(p.status, DEV_NONFINITE);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PARTS; k++) amax = fmaxf(amax, s_amax[k][combo]);
    const float scale = fmaxf(q8_scale<kFmt>(amax), old_scale);
    const float div = scale > 0.0f ? scale : 1.0f;
    unsigned char* base = (is_v ? p.map.v_pool : p.map.k_pool) + (size_t)id * p.map.block_stride + kvh * HD;
    if (scale > old_scale) {  // slots before the segment move to the larger scale
        for (uint32_t t = part; t < slot0; t += PARTS) {
            uint32_t* at = reinterpret_cast<uint32_t*>(base + (size_t)t * Q8_ROW_BYTES) + lane;
            const uint32_t w = __ldcg(at);
            uint32_t o = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) o |= q8_code<kFmt>(q8_value<kFmt>((w >> (8 * j)) & 0xffu) * old_scale, div) << (8 * j);
            *at = o;
        }
    }
    auto store_row = [&](uint32_t i, const float (&x)[4]) {
        uint16_t* at = reinterpret_cast<uint16_t*>(base + (size_t)(slot0 + i) * Q8_ROW_BYTES);
        at[lane] = (uint16_t)(q8_code<kFmt>(x[0], div) | (q8_code<kFmt>(x[1], div) << 8));
        at[32 + lane] = (uint16_t)(q8_code<kFmt>(x[2], div) | (q8_code<kFmt>(x[3], div) << 8));
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const uint32_t i = part + k * PARTS;
        if (i < n) store_row(i, keep[k]);
    }
    for (uint32_t i = part + KEEP * PARTS; i < n; i += PARTS) {
        float x[4];
        load_row(i, x);
        store_row(i, x);
    }
    if (part == 0 && lane == 0) *scale_at = scale;
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
    return launch_pdl(format == Q8_INT8 ? append_q8_kernel<Q8_INT8> : append_q8_kernel<Q8_E4M3>, dim3(rows), dim3(aq::THREADS), 0,
                      stream, p);
}

}  // namespace oxi
