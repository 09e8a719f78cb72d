// Storing into and reading from the packed key/value cache (format: kv4.cuh).
//
//   rope_store_kv4   per token row [queries | keys | values]: queries rotated, keys rotated, rounded to the engine's type and packed,
//                    values packed, both into their page.  The row may still be the k-split partial sums of its product.
//   kv4_read         rows of the cache back as numbers (float32 or bfloat16).
//
// Rotation: lo = a cos - b sin, hi = b cos + a sin over the pairs (i, i + rotary_dim / 2), products and sums rounded one by one (no
// fused multiply-add: the stored codes shall not depend on how a compiler contracts).
#include "kv4.cuh"

namespace {

// Eight neighbouring numbers.
struct Eight { float x[8]; };
template <typename T> struct Row;
template <> struct Row<float> {
    static __device__ __forceinline__ Eight load(const float* p) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
    static __device__ __forceinline__ void store(float* p, const Eight& v) {
        *reinterpret_cast<float4*>(p) = make_float4(v.x[0], v.x[1], v.x[2], v.x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v.x[4], v.x[5], v.x[6], v.x[7]);
    }
    static __device__ __forceinline__ float rounded(float v) { return v; }
};
template <> struct Row<__nv_bfloat16> {
    static __device__ __forceinline__ Eight load(const __nv_bfloat16* p) {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        Eight v;
#pragma unroll
        for (int i = 0; i < 4; ++i) { v.x[2 * i] = __uint_as_float(w[i] << 16); v.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        return v;
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const Eight& v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v.x[2 * i], v.x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float rounded(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
};

__device__ __forceinline__ float rot_lo(float a, float b, float c, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
__device__ __forceinline__ float rot_hi(float a, float b, float c, float s) { return __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)); }
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

struct Kv4StoreArgs {
    const void* rows;          // [tokens][row_width] of T, or null: `parts`
    const float* parts;        // [splits][tokens][row_width] float32
    int splits;
    size_t split_stride;
    void* q_out;               // rotated queries: row t at t * q_stride (may be `rows` itself)
    size_t q_stride;
    const float* cos_table;    // [tokens][rotary_dim / 2]; null: nothing is rotated
    const float* sin_table;
    const int* slots;          // [tokens], < 0: not stored; null: queries only
    uint8_t* cache;
    int heads, kv_heads, head_dim, rotary_dim, page_size;
    int q_warps, warps;        // of a token: warps that rotate queries, and all
};

template <typename T, bool PARTS>
__device__ __forceinline__ Eight row_eight(const Kv4StoreArgs& a, size_t at) {
    if constexpr (PARTS) {
        const float4 u = sum_parts4(a.parts + at, a.splits, a.split_stride), v = sum_parts4(a.parts + at + 4, a.splits, a.split_stride);
        return {{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w}};
    } else {
        return Row<T>::load(static_cast<const T*>(a.rows) + at);
    }
}

__device__ __forceinline__ float min3(float a, float b, float c) {
    float y;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Packs 32 numbers held by 4 neighbouring lanes, eight each (all lanes of the warp call): the lane's code word, the group's (s, z), and
// whether anything of the lane's, or s or z, or the number of the top code, is not finite.  (s may be rounded up, by 2^-8 of it: float32
// numbers next to the largest one would come back as infinity.)
//
// Four instructions a number, for this is where the kernel's instructions go: x - z, times r, plus 1.5 2^23 (whose last bit counts 1: the
// sum's low bits are the product rounded to the nearest even), and a multiply-add that shifts those bits into the word; what the
// addends have on top is taken off all at once.  No code needs a clamp: x >= z, and (max - z) r <= 15 (1 + 2^-8) with s a normal number.
__device__ __forceinline__ void pack_group(const Eight& v, uint32_t& word, uint32_t& par, bool& bad) {
    const float* x = v.x;
    float lo = min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), fminf(x[6], x[7]));
    float hi = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7]));
    float zeros = 0.f;                                  // NaN if a number is not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) zeros = fmaf(x[i], 0.f, zeros);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float z = __bfloat162float(__float2bfloat16_rd(lo));
    float s = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f)));
    if (s < 1.17549435e-38f) s = 0.f;
    bad = zeros != 0.f || !finite(fmaf(15.f, s, z));     // (which z or s that is not finite makes NaN or infinite too)
    const float r = s > 0.f ? __frcp_rn(s) : 0.f;
    constexpr uint32_t kOnTop = 0x4b400000u;            // 1.5 2^23
    word = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) word += (__float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[i], z), r), 12582912.f)) - kOnTop) << kv4_bit(i);
    par = __float_as_uint(s) >> 16 | (__float_as_uint(z) & 0xffff0000u);
}

// grid (tokens, blocks of a token's warps).  A thread works on eight neighbouring numbers with 16-byte loads and stores.  Bound by
// latency for a few rows (8 rows of 48 heads of 128: 2.5 us back to back; in place from 2, 4 or 8 partial sums, as a decode step stores
// them, 3.5, 3.8 and 4.8); for many by the latency of a row's loads over the rows that
// run at a time, half of memory's rate: 2048 rows (45 MB) 14.0 us, 8192 rows 46.8 us.  Five blocks an SM rather than four: 46.8 instead of
// 51.2 us.  Four numbers a thread took 59.7 us, a loop over rows with the next row's numbers held in registers 106 us.
template <typename T, bool PARTS>
__global__ void __launch_bounds__(384, sizeof(T) == 2 && !PARTS ? 5 : 1)
rope_store_kv4_kernel(const Kv4StoreArgs a) {
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, D = a.head_dim, half = a.rotary_dim / 2, lane = threadIdx.x & 31;
    const int warp = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const size_t row = (size_t)t * ((size_t)(a.heads + 2 * a.kv_heads) * D);
    const float* cs = a.cos_table + (size_t)t * half;
    const float* sn = a.sin_table + (size_t)t * half;
    if (warp < a.q_warps) {
        // ---- queries: the two halves of a pair by one thread (they may be rotated in place) --------------------------------
        const int pairs = half / 8, per_head = pairs + (D - a.rotary_dim) / 8, w = warp * 32 + lane;
        if (w >= a.heads * per_head) return;
        const int h = w / per_head, j = w - h * per_head;
        T* to = static_cast<T*>(a.q_out) + (size_t)t * a.q_stride + (size_t)h * D;
        if (j >= pairs) {
            const int c = a.rotary_dim + (j - pairs) * 8;
            Row<T>::store(to + c, row_eight<T, PARTS>(a, row + (size_t)h * D + c));
            return;
        }
        const int c = j * 8;
        const Eight x = row_eight<T, PARTS>(a, row + (size_t)h * D + c), y = row_eight<T, PARTS>(a, row + (size_t)h * D + c + half);
        const Eight co = Row<float>::load(cs + c), si = Row<float>::load(sn + c);
        Eight lo, hi;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo.x[i] = rot_lo(x.x[i], y.x[i], co.x[i], si.x[i]);
            hi.x[i] = rot_hi(x.x[i], y.x[i], co.x[i], si.x[i]);
        }
        Row<T>::store(to + c, lo);
        Row<T>::store(to + c + half, hi);
        return;
    }
    if (warp >= a.warps) return;
    // ---- keys and values: a head is spread over 4, 8, 16 or 32 lanes of one warp ---------------------------------------------
    const int slot = a.slots[t];
    if (slot < 0) return;
    const int G = D / 32, lanes = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
    const int sub = lane / lanes, c = 8 * (lane - sub * lanes), g = (warp - a.q_warps) * (32 / lanes) + sub;
    const bool here = g < a.kv_heads && c < D;
    Eight k, v;
#pragma unroll
    for (int i = 0; i < 8; ++i) k.x[i] = v.x[i] = 0.f;
    if (here) {
        const size_t kat = row + (size_t)(a.heads + g) * D + c;
        k = row_eight<T, PARTS>(a, kat);
        v = row_eight<T, PARTS>(a, kat + (size_t)a.kv_heads * D);
        if (c < half) {
            const Eight y = row_eight<T, PARTS>(a, kat + half), co = Row<float>::load(cs + c), si = Row<float>::load(sn + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) k.x[i] = rot_lo(k.x[i], y.x[i], co.x[i], si.x[i]);
        } else if (c < a.rotary_dim) {
            const Eight x = row_eight<T, PARTS>(a, kat - half), co = Row<float>::load(cs + c - half), si = Row<float>::load(sn + c - half);
#pragma unroll
            for (int i = 0; i < 8; ++i) k.x[i] = rot_hi(x.x[i], k.x[i], co.x[i], si.x[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k.x[i] = Row<T>::rounded(k.x[i]);
            if (PARTS) v.x[i] = Row<T>::rounded(v.x[i]);
        }
    }
    uint32_t kw, kp, vw, vp;
    bool bk, bv;
    pack_group(k, kw, kp, bk);
    pack_group(v, vw, vp, bv);
    const uint32_t head_lanes = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (sub * lanes);
    const bool bad = (__ballot_sync(0xffffffffu, bk || bv) & head_lanes) != 0;
    if (!here) return;
    const int page = slot / a.page_size, off = slot - page * a.page_size, grp = c / 32, j = (c % 32) / 8;
    uint8_t* block = a.cache + ((size_t)page * a.kv_heads + g) * kv4_block_bytes(a.page_size, G);
    uint16_t* vc = reinterpret_cast<uint16_t*>(block + kv4_value_codes(a.page_size, G) + (size_t)off * 16 * G);
    reinterpret_cast<uint32_t*>(block + (size_t)off * 16 * G)[j * G + grp] = bad ? 0u : kw;
    vc[2 * j * G + grp] = (uint16_t)(bad ? 0u : vw & 0xffffu);
    vc[(2 * j + 1) * G + grp] = (uint16_t)(bad ? 0u : vw >> 16);
    if (j == 0) {
        reinterpret_cast<uint32_t*>(block + kv4_key_par(a.page_size, G) + (size_t)off * 4 * G)[grp] = bad ? 0x7fc07fc0u : kp;
        reinterpret_cast<uint32_t*>(block + kv4_value_par(a.page_size, G) + (size_t)off * 4 * G)[grp] = bad ? 0u : vp;
    }
}

// out[n][2][kv_heads][D] of the slots' keys and values: a thread per word of eight numbers.  A slot below 0 reads as zeros.  Bound by
// the latency of slot -> word -> store, for many slots too (2048 slots of 8 heads of 128 to float32, 19 MB, 5.6 us, 3.0 at the rate of a
// copy; 8192 slots 19.1 us, 62% of that rate); a block a slot took 30.6 us there.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slots, T* __restrict__ out, unsigned total, int kv_heads, int head_dim,
                int page_size) {
    pdl_trigger();
    pdl_wait();
    const unsigned w = blockIdx.x * 256 + threadIdx.x;
    if (w >= total) return;
    const unsigned G = head_dim / 32, words = 4 * G, line = w / words, u = w - line * words;       // eight numbers u * 8 .. of the head
    const unsigned i = line / (2 * kv_heads), rest = line - i * 2 * kv_heads;
    const bool value = rest >= (unsigned)kv_heads;
    const unsigned h = value ? rest - kv_heads : rest, g = u / 4, j = u % 4;
    const int slot = slots[i];
    Eight x = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
    if (slot >= 0) {
        const int page = slot / page_size, off = slot - page * page_size;
        const uint8_t* block = cache + ((size_t)page * kv_heads + h) * kv4_block_bytes(page_size, G);
        uint32_t word, par;
        if (!value) {
            word = reinterpret_cast<const uint32_t*>(block + off * 16 * G)[j * G + g];
            par = reinterpret_cast<const uint32_t*>(block + kv4_key_par(page_size, G) + off * 4 * G)[g];
        } else {
            const uint16_t* v = reinterpret_cast<const uint16_t*>(block + kv4_value_codes(page_size, G) + off * 16 * G);
            word = (uint32_t)v[2 * j * G + g] | (uint32_t)v[(2 * j + 1) * G + g] << 16;
            par = reinterpret_cast<const uint32_t*>(block + kv4_value_par(page_size, G) + off * 4 * G)[g];
        }
        const float s = kv4_step(par), z = kv4_zero(par);
#pragma unroll
        for (int e = 0; e < 8; ++e) x.x[e] = fmaf(s, (float)((word >> kv4_bit(e)) & 15u), z);
    }
    Row<T>::store(out + (size_t)w * 8, x);
}

}  // namespace

// rows: [tokens, (heads + 2 kv_heads) * head_dim] of `dtype`, or null with `parts` [splits][tokens][the same] float32.  q_out: where
// the rotated queries go, rows q_stride numbers apart (the rows themselves: in place).  cos / sin [tokens, rotary_dim / 2]; slots
// null: nothing is stored.  Every pointer on a 16-byte boundary.
LLM_API int llm_rope_store_kv4(const void* rows, const float* parts, int splits, long long split_stride, void* q_out, long long q_stride,
                               const float* cos_table, const float* sin_table, const int* slots, void* cache, int dtype, int tokens, int heads,
                               int kv_heads, int head_dim, int rotary_dim, int page_size, cudaStream_t stream) {
    if (tokens == 0) return 0;
    if (!kv4_geometry(head_dim, slots ? page_size : 4))
        LLM_FAIL(-1, "rope_store_kv4: head_dim %d must be a multiple of 32 up to %d and page_size %d a multiple of 4", head_dim, kKv4MaxDim,
                 page_size);
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16) LLM_FAIL(-1, "rope_store_kv4: rotary_dim %d must be a multiple of 16 up to head_dim %d", rotary_dim, head_dim);
    if (rotary_dim && (!cos_table || !sin_table)) LLM_FAIL(-1, "rope_store_kv4: a rotation needs its tables");
    if (!rows && (splits < 1 || splits > kMaxParts || split_stride % 4)) LLM_FAIL(-1, "rope_store_kv4: 1..%d splits (%d), a stride that is a multiple of 4", kMaxParts, splits);
    if (heads <= 0 || kv_heads <= 0) LLM_FAIL(-1, "rope_store_kv4: heads %d / kv_heads %d", heads, kv_heads);
    Kv4StoreArgs a;
    a.rows = rows; a.parts = parts; a.splits = splits; a.split_stride = (size_t)split_stride;
    a.q_out = q_out; a.q_stride = (size_t)q_stride;
    a.cos_table = cos_table; a.sin_table = sin_table; a.slots = slots; a.cache = (uint8_t*)cache;
    a.heads = heads; a.kv_heads = kv_heads; a.head_dim = head_dim; a.rotary_dim = rotary_dim; a.page_size = page_size;
    const int per_head = rotary_dim / 16 + (head_dim - rotary_dim) / 8;
    // queries that stay where they are and are not rotated have nothing to be done to them
    const bool idle = rotary_dim == 0 && rows != nullptr && q_out == rows;
    a.q_warps = idle ? 0 : (heads * per_head + 31) / 32;
    const int heads_per_warp = head_dim <= 32 ? 8 : head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1;
    a.warps = a.q_warps + (slots ? (kv_heads + heads_per_warp - 1) / heads_per_warp : 0);
    if (a.warps == 0) return 0;
    const int per_block = a.warps < 12 ? a.warps : 12, blocks = (a.warps + per_block - 1) / per_block;
    if (blocks > 65535) LLM_FAIL(-1, "rope_store_kv4: too many heads");
    return llm_dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        if (rows) llm_launch(rope_store_kv4_kernel<T, false>, dim3(tokens, blocks), 32 * per_block, 0, stream, a);
        else llm_launch(rope_store_kv4_kernel<T, true>, dim3(tokens, blocks), 32 * per_block, 0, stream, a);
        LLM_CHECK_LAUNCH("rope_store_kv4");
        return 0;
    });
}

// out [n, 2, kv_heads, head_dim] of `dtype`.
LLM_API int llm_kv4_read(const void* cache, const int* slots, void* out, int dtype, int n, int kv_heads, int head_dim, int page_size,
                         cudaStream_t stream) {
    if (n == 0) return 0;
    if (!kv4_geometry(head_dim, page_size) || kv_heads <= 0)
        LLM_FAIL(-1, "kv4_read: head_dim %d must be a multiple of 32 up to %d and page_size %d a multiple of 4", head_dim, kKv4MaxDim, page_size);
    return llm_dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        const long long words = (long long)n * 2 * kv_heads * (head_dim / 8);
        if (words > 0xffff0000ll) LLM_FAIL(-1, "kv4_read: too many rows");
        llm_launch(kv4_read_kernel<T>, dim3((unsigned)((words + 255) / 256)), 256, 0, stream, (const uint8_t*)cache, slots, (T*)out, (unsigned)words,
                   kv_heads, head_dim, page_size);
        LLM_CHECK_LAUNCH("kv4_read");
        return 0;
    });
}

LLM_TRACE_EXPORT(kv4_store)
