// Attention of single rows over 8-bit paged caches and, with a sliding window and sinks, over f16 caches:
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(q.k_t / sqrt(128)),  t < len and (t >= len - window or t < sinks)
// A CTA takes one row and one KV head, a warp one query head of its group; a lane holds 4 of the 128 dims and
// the running maximum and sum are kept per warp.
#include "kernels.h"
#include "q8.cuh"

namespace oxi {

struct F16Rows {
    const uint64_t* k_ptrs;
    const uint64_t* v_ptrs;
    PagedMap map;
    const uint32_t* row_seq;
    uint64_t k, v, trow;
    bool paged;
    __device__ uint32_t begin(uint32_t r, uint32_t len, int) {
        paged = map.block_tables != nullptr;
        if (paged) {
            trow = (uint64_t)(row_seq ? row_seq[r] : r) * map.max_blocks;
            return ((len - 1u) >> map.lbs) >= map.max_blocks ? DEV_BAD_SEQ_LEN : 0u;
        }
        k = k_ptrs[r];
        v = v_ptrs[r];
        return ((k | v) & 15ull) ? DEV_MISALIGNED_PTR : 0u;
    }
    __device__ uint32_t load(uint32_t t, int kvh, int lane, float (&kx)[4], float (&vx)[4]) {
        uint32_t bad = 0;
        size_t off = (size_t)t * KV_ROW_BYTES;
        const unsigned char *kb = (const unsigned char*)k, *vb = (const unsigned char*)v;
        if (paged) {
            uint32_t id = map.block_tables[trow + (t >> map.lbs)];
            if (id >= map.num_blocks) {
                bad = DEV_BAD_BLOCK;
                id = 0;
            }
            off = (size_t)id * map.block_stride + (size_t)(t & ((1u << map.lbs) - 1u)) * KV_ROW_BYTES;
            kb = map.k_pool;
            vb = map.v_pool;
        }
        off += kvh * HD * 2;
        const uint2 a = reinterpret_cast<const uint2*>(kb + off)[lane], b = reinterpret_cast<const uint2*>(vb + off)[lane];
        const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            kx[2 * i] = h2f((uint16_t)w[i]);
            kx[2 * i + 1] = h2f((uint16_t)(w[i] >> 16));
            vx[2 * i] = h2f((uint16_t)w[2 + i]);
            vx[2 * i + 1] = h2f((uint16_t)(w[2 + i] >> 16));
        }
        return bad;
    }
};

template <uint32_t kFmt>
struct Q8Rows {
    Q8Map map;
    const uint32_t* row_seq;
    uint64_t trow;
    __device__ uint32_t begin(uint32_t r, uint32_t len, int) {
        trow = (uint64_t)(row_seq ? row_seq[r] : r) * map.max_blocks;
        return ((len - 1u) >> map.lbs) >= map.max_blocks ? DEV_BAD_SEQ_LEN : 0u;
    }
    __device__ uint32_t load(uint32_t t, int kvh, int lane, float (&kx)[4], float (&vx)[4]) {
        uint32_t bad = 0;
        uint32_t id = map.block_tables[trow + (t >> map.lbs)];
        if (id >= map.num_blocks) {
            bad = DEV_BAD_BLOCK;
            id = 0;
        }
        const size_t off = (size_t)id * map.block_stride + (size_t)(t & ((1u << map.lbs) - 1u)) * Q8_ROW_BYTES + kvh * HD;
        const uint32_t a = reinterpret_cast<const uint32_t*>(map.k_pool + off)[lane], b = reinterpret_cast<const uint32_t*>(map.v_pool + off)[lane];
        const float ks = map.k_scales[(size_t)id * map.scale_stride + kvh], vs = map.v_scales[(size_t)id * map.scale_stride + kvh];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            kx[i] = q8_value<kFmt>((a >> (8 * i)) & 0xffu) * ks;
            vx[i] = q8_value<kFmt>((b >> (8 * i)) & 0xffu) * vs;
        }
        return bad;
    }
};

template <class KV>
__global__ void __launch_bounds__(128)
attn_rows_kernel(uint16_t* ctx_out, const uint16_t* q, const uint16_t* gate, KV kv, const uint32_t* seq_lens, uint32_t window,
                 uint32_t sinks, uint32_t max_seq_len, uint32_t* status) {
    const uint32_t r = blockIdx.x >> 2;
    const int kvh = blockIdx.x & 3, lane = threadIdx.x & 31, head = kvh * 4 + (threadIdx.x >> 5);
    pdl_wait();
    const uint32_t len = seq_lens[r];
    uint32_t bad = len == 0u || len > max_seq_len ? DEV_BAD_SEQ_LEN : 0u;
    if (!bad) bad = kv.begin(r, len, kvh);
    if (bad) {
        if (threadIdx.x == 0) atomicOr(status, bad);
        return;
    }
    const uint32_t start = window_start(len, window);
    const size_t rh = ((size_t)r * NQ + head) * HD;
    float qx[4];
    const uint2 a = reinterpret_cast<const uint2*>(q + rh)[lane];
    qx[0] = h2f((uint16_t)a.x);
    qx[1] = h2f((uint16_t)(a.x >> 16));
    qx[2] = h2f((uint16_t)a.y);
    qx[3] = h2f((uint16_t)(a.y >> 16));
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t t = sinks < start && sinks ? 0u : (sinks ? 0u : start); t < len; t++) {
        if (t >= sinks && t < start) t = start;
        float kx[4], vx[4];
        bad |= kv.load(t, kvh, lane, kx, vx);
        float x = qx[0] * kx[0] + qx[1] * kx[1] + qx[2] * kx[2] + qx[3] * kx[3];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
        x *= ATTN_SCALE * LOG2E;
        const float mn = fmaxf(m, x), corr = exp2f(m - mn), pr = exp2f(x - mn);
        m = mn;
        l = l * corr + pr;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * corr + pr * vx[i];
    }
    if (bad && threadIdx.x == 0) atomicOr(status, bad);
    const float f = (gate ? sigmoid_ref(h2f(gate[(size_t)r * NQ + head])) : 1.0f) / l;
    reinterpret_cast<uint2*>(ctx_out + rh)[lane] = make_uint2(pack_h2(o[0] * f, o[1] * f), pack_h2(o[2] * f, o[3] * f));
}

cudaError_t launch_attn_q8(cudaStream_t stream, void* ctx_out, const void* q, const void* gate, const Q8Map& map, uint32_t format,
                           const uint32_t* row_seq, const uint32_t* seq_lens, uint32_t rows, uint32_t window, uint32_t sinks,
                           uint32_t max_seq_len, uint32_t* status) {
    if (format == Q8_INT8) {
        Q8Rows<Q8_INT8> kv{map, row_seq, 0};
        return launch_pdl(attn_rows_kernel<Q8Rows<Q8_INT8>>, dim3(rows * 4), dim3(128), 0, stream, (uint16_t*)ctx_out, (const uint16_t*)q,
                          (const uint16_t*)gate, kv, seq_lens, window, sinks, max_seq_len, status);
    }
    Q8Rows<Q8_E4M3> kv{map, row_seq, 0};
    return launch_pdl(attn_rows_kernel<Q8Rows<Q8_E4M3>>, dim3(rows * 4), dim3(128), 0, stream, (uint16_t*)ctx_out, (const uint16_t*)q,
                      (const uint16_t*)gate, kv, seq_lens, window, sinks, max_seq_len, status);
}

cudaError_t launch_attn_sinks(cudaStream_t stream, void* ctx_out, const void* q, const void* gate, const uint64_t* k_ptrs,
                              const uint64_t* v_ptrs, const PagedMap* pm, const uint32_t* row_seq, const uint32_t* seq_lens,
                              uint32_t rows, uint32_t window, uint32_t sinks, uint32_t max_seq_len, uint32_t* status) {
    F16Rows kv{k_ptrs, v_ptrs, pm ? *pm : PagedMap{}, row_seq, 0, 0, 0, false};
    return launch_pdl(attn_rows_kernel<F16Rows>, dim3(rows * 4), dim3(128), 0, stream, (uint16_t*)ctx_out, (const uint16_t*)q,
                      (const uint16_t*)gate, kv, seq_lens, window, sinks, max_seq_len, status);
}

}  // namespace oxi
