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

template <typename T> struct Quad;
template <> struct Quad<float> {
    static __device__ __forceinline__ float4 load(const float* p) { return *reinterpret_cast<const float4*>(p); }
    static __device__ __forceinline__ void store(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
    static __device__ __forceinline__ float rounded(float v) { return v; }
};
template <> struct Quad<__nv_bfloat16> {
    static __device__ __forceinline__ float4 load(const __nv_bfloat16* p) {
        const uint2 raw = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                           __uint_as_float(raw.y & 0xffff0000u));
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, float4 v) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
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
    int q_blocks;              // blocks along y that rotate queries; the others pack keys and values
};

template <typename T, bool PARTS>
__device__ __forceinline__ float4 row_quad(const Kv4StoreArgs& a, size_t at) {
    if constexpr (PARTS) return sum_parts4(a.parts + at, a.splits, a.split_stride);
    else return Quad<T>::load(static_cast<const T*>(a.rows) + at);
}

// Packs 32 numbers held by 8 neighbouring lanes, four each (all lanes of the warp call): the lane's four codes at their bits of an
// 8-number word that it shares with its neighbour, the group's (s, z), and whether anything is not finite.
__device__ __forceinline__ void pack_group(float4 x, int lane, uint32_t& word, uint32_t& par, bool& bad) {
    float lo = fminf(fminf(x.x, x.y), fminf(x.z, x.w)), hi = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float z = __bfloat162float(__float2bfloat16_rd(lo));
    float s = __bfloat162float(__float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, z), 1.0f / 15.0f)));
    if (s < 1.17549435e-38f) s = 0.f;
    bad = !(finite(x.x) && finite(x.y) && finite(x.z) && finite(x.w) && finite(z) && finite(s));
    const float r = s > 0.f ? __frcp_rn(s) : 0.f;
    auto code = [&](float v) { return (uint32_t)(int)fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(v, z), r)), 0.f), 15.f); };
    const uint32_t quad = code(x.x) | code(x.y) << 16 | code(x.z) << 4 | code(x.w) << 20;
    word = quad << (8 * (lane & 1));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    par = __float_as_uint(s) >> 16 | (__float_as_uint(z) & 0xffff0000u);
}

// grid (tokens, q_blocks + blocks of key/value heads), 256 threads.  QUADS: four-number pieces a lane holds of a head (a head is
// spread over 8, 16 or 32 lanes of one warp, head_dim / 4 pieces in all).
template <typename T, bool PARTS, int QUADS>
__global__ void __launch_bounds__(256)
rope_store_kv4_kernel(const Kv4StoreArgs a) {
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, D = a.head_dim, half = a.rotary_dim / 2;
    const size_t row = (size_t)t * ((size_t)(a.heads + 2 * a.kv_heads) * D);
    const float* cs = a.cos_table + (size_t)t * half;
    const float* sn = a.sin_table + (size_t)t * half;
    if ((int)blockIdx.y < a.q_blocks) {
        // ---- queries: the two halves of a pair by one thread (they may be rotated in place) --------------------------------
        const int pairs = half / 4, rest = (D - a.rotary_dim) / 4, per_head = pairs + rest;
        const int w = blockIdx.y * 256 + threadIdx.x;
        if (w >= a.heads * per_head) return;
        const int h = w / per_head, j = w - h * per_head;
        T* to = static_cast<T*>(a.q_out) + (size_t)t * a.q_stride + (size_t)h * D;
        if (j >= pairs) {
            const int c = a.rotary_dim + (j - pairs) * 4;
            Quad<T>::store(to + c, row_quad<T, PARTS>(a, row + (size_t)h * D + c));
            return;
        }
        const int c = j * 4;
        const float4 x = row_quad<T, PARTS>(a, row + (size_t)h * D + c), y = row_quad<T, PARTS>(a, row + (size_t)h * D + c + half);
        const float4 co = *reinterpret_cast<const float4*>(cs + c), si = *reinterpret_cast<const float4*>(sn + c);
        Quad<T>::store(to + c, make_float4(rot_lo(x.x, y.x, co.x, si.x), rot_lo(x.y, y.y, co.y, si.y), rot_lo(x.z, y.z, co.z, si.z),
                                           rot_lo(x.w, y.w, co.w, si.w)));
        Quad<T>::store(to + c + half, make_float4(rot_hi(x.x, y.x, co.x, si.x), rot_hi(x.y, y.y, co.y, si.y), rot_hi(x.z, y.z, co.z, si.z),
                                                  rot_hi(x.w, y.w, co.w, si.w)));
        return;
    }
    // ---- keys and values ---------------------------------------------------------------------------------------------------
    const int slot = a.slots[t];
    if (slot < 0) return;
    const int lane = threadIdx.x & 31, G = D / 32;
    const int lanes = D == 32 ? 8 : D == 64 ? 16 : 32;                   // lanes of a head
    const int sub = lane / lanes, at = lane - sub * lanes;
    const int g = ((blockIdx.y - a.q_blocks) * 8 + (threadIdx.x >> 5)) * (32 / lanes) + sub;
    const bool here = g < a.kv_heads;
    uint32_t kw[QUADS], kp[QUADS], vw[QUADS], vp[QUADS];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        const int c = 4 * at + 128 * i;
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (here && c < D) {
            const size_t kat = row + (size_t)(a.heads + g) * D, vat = kat + (size_t)a.kv_heads * D;
            k = row_quad<T, PARTS>(a, kat + c);
            if (c < half) {
                const float4 y = row_quad<T, PARTS>(a, kat + c + half);
                const float4 co = *reinterpret_cast<const float4*>(cs + c), si = *reinterpret_cast<const float4*>(sn + c);
                k = make_float4(rot_lo(k.x, y.x, co.x, si.x), rot_lo(k.y, y.y, co.y, si.y), rot_lo(k.z, y.z, co.z, si.z),
                                rot_lo(k.w, y.w, co.w, si.w));
            } else if (c < a.rotary_dim) {
                const float4 x = row_quad<T, PARTS>(a, kat + c - half);
                const float4 co = *reinterpret_cast<const float4*>(cs + c - half), si = *reinterpret_cast<const float4*>(sn + c - half);
                k = make_float4(rot_hi(x.x, k.x, co.x, si.x), rot_hi(x.y, k.y, co.y, si.y), rot_hi(x.z, k.z, co.z, si.z),
                                rot_hi(x.w, k.w, co.w, si.w));
            }
            v = row_quad<T, PARTS>(a, vat + c);
            k = make_float4(Quad<T>::rounded(k.x), Quad<T>::rounded(k.y), Quad<T>::rounded(k.z), Quad<T>::rounded(k.w));
            v = make_float4(Quad<T>::rounded(v.x), Quad<T>::rounded(v.y), Quad<T>::rounded(v.z), Quad<T>::rounded(v.w));
        }
        bool bk, bv;
        pack_group(k, lane, kw[i], kp[i], bk);
        pack_group(v, lane, vw[i], vp[i], bv);
        bad = bad || bk || bv;
    }
    const uint32_t head_lanes = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (sub * lanes);
    bad = (__ballot_sync(0xffffffffu, bad) & head_lanes) != 0;
    if (!here) return;
    const int page = slot / a.page_size, off = slot - page * a.page_size;
    uint8_t* block = a.cache + ((size_t)page * a.kv_heads + g) * kv4_block_bytes(a.page_size, G);
    uint32_t* kc = reinterpret_cast<uint32_t*>(block + (size_t)off * 16 * G);
    uint32_t* kpar = reinterpret_cast<uint32_t*>(block + kv4_key_par(a.page_size, G) + (size_t)off * 4 * G);
    uint16_t* vc = reinterpret_cast<uint16_t*>(block + kv4_value_codes(a.page_size, G) + (size_t)off * 16 * G);
    uint32_t* vpar = reinterpret_cast<uint32_t*>(block + kv4_value_par(a.page_size, G) + (size_t)off * 4 * G);
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        const int c = 4 * at + 128 * i;
        if (c >= D) break;
        const int grp = c / 32, j = (c % 32) / 8;
        if (lane & 1) {
            vc[2 * j * G + grp] = (uint16_t)(bad ? 0u : vw[i] & 0xffffu);
            vc[(2 * j + 1) * G + grp] = (uint16_t)(bad ? 0u : vw[i] >> 16);
        } else {
            kc[j * G + grp] = bad ? 0u : kw[i];
        }
        if ((at & 7) == 0) {
            kpar[grp] = bad ? 0x7fc07fc0u : kp[i];
            vpar[grp] = bad ? 0u : vp[i];
        }
    }
}

// out[n][2][kv_heads][D] of the slots' keys and values: a thread per word of eight numbers.  A slot below 0 reads as zeros.
template <typename T>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ slots, T* __restrict__ out, int n, int kv_heads, int head_dim,
                int page_size) {
    pdl_trigger();
    pdl_wait();
    const int G = head_dim / 32, words = 4 * G;
    const long long w = (long long)blockIdx.x * 256 + threadIdx.x;
    if (w >= (long long)n * 2 * kv_heads * words) return;
    const int u = (int)(w % words);                       // eight numbers u * 8 .. of the head
    const long long rest = w / words;
    const int h = (int)(rest % kv_heads), which = (int)(rest / kv_heads % 2), i = (int)(rest / (2 * kv_heads));
    const int slot = slots[i], g = u / 4, j = u % 4;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0) {
        const int page = slot / page_size, off = slot - page * page_size;
        const uint8_t* block = cache + ((size_t)page * kv_heads + h) * kv4_block_bytes(page_size, G);
        uint32_t word, par;
        if (which == 0) {
            word = reinterpret_cast<const uint32_t*>(block + (size_t)off * 16 * G)[j * G + g];
            par = reinterpret_cast<const uint32_t*>(block + kv4_key_par(page_size, G) + (size_t)off * 4 * G)[g];
        } else {
            const uint16_t* v = reinterpret_cast<const uint16_t*>(block + kv4_value_codes(page_size, G) + (size_t)off * 16 * G);
            word = (uint32_t)v[2 * j * G + g] | (uint32_t)v[(2 * j + 1) * G + g] << 16;
            par = reinterpret_cast<const uint32_t*>(block + kv4_value_par(page_size, G) + (size_t)off * 4 * G)[g];
        }
        const float s = kv4_step(par), z = kv4_zero(par);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(s, (float)((word >> kv4_bit(e)) & 15u), z);
    }
    T* to = out + (size_t)w * 8;
    Quad<T>::store(to, make_float4(x[0], x[1], x[2], x[3]));
    Quad<T>::store(to + 4, make_float4(x[4], x[5], x[6], x[7]));
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
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 8) LLM_FAIL(-1, "rope_store_kv4: rotary_dim %d must be a multiple of 8 up to head_dim %d", rotary_dim, head_dim);
    if (rotary_dim && (!cos_table || !sin_table)) LLM_FAIL(-1, "rope_store_kv4: a rotation needs its tables");
    if (!rows && (splits < 1 || splits > kMaxParts || split_stride % 4)) LLM_FAIL(-1, "rope_store_kv4: 1..%d splits (%d), a stride that is a multiple of 4", kMaxParts, splits);
    if (heads <= 0 || kv_heads <= 0) LLM_FAIL(-1, "rope_store_kv4: heads %d / kv_heads %d", heads, kv_heads);
    Kv4StoreArgs a;
    a.rows = rows; a.parts = parts; a.splits = splits; a.split_stride = (size_t)split_stride;
    a.q_out = q_out; a.q_stride = (size_t)q_stride;
    a.cos_table = cos_table; a.sin_table = sin_table; a.slots = slots; a.cache = (uint8_t*)cache;
    a.heads = heads; a.kv_heads = kv_heads; a.head_dim = head_dim; a.rotary_dim = rotary_dim; a.page_size = page_size;
    const int per_head = rotary_dim / 8 + (head_dim - rotary_dim) / 4;
    // queries that stay where they are and are not rotated have nothing to be done to them
    const bool idle = rotary_dim == 0 && rows != nullptr && q_out == rows;
    a.q_blocks = idle ? 0 : (heads * per_head + 255) / 256;
    const int per_warp = head_dim == 32 ? 4 : head_dim == 64 ? 2 : 1;
    const int kv_blocks = slots ? (kv_heads + 8 * per_warp - 1) / (8 * per_warp) : 0;
    if (a.q_blocks + kv_blocks == 0) return 0;
    if (a.q_blocks + kv_blocks > 65535) LLM_FAIL(-1, "rope_store_kv4: too many heads");
    const dim3 grid(tokens, a.q_blocks + kv_blocks);
    return llm_dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        auto go = [&](auto kernel) { llm_launch(kernel, grid, 256, 0, stream, a); };
        if (rows) { if (head_dim <= 128) go(rope_store_kv4_kernel<T, false, 1>); else go(rope_store_kv4_kernel<T, false, 2>); }
        else { if (head_dim <= 128) go(rope_store_kv4_kernel<T, true, 1>); else go(rope_store_kv4_kernel<T, true, 2>); }
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
    const long long blocks = ((long long)n * 2 * kv_heads * (head_dim / 8) + 255) / 256;
    if (blocks > 0x7fffffffll) LLM_FAIL(-1, "kv4_read: too many rows");
    return llm_dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        llm_launch(kv4_read_kernel<T>, dim3((unsigned)blocks), 256, 0, stream, (const uint8_t*)cache, slots, (T*)out, n, kv_heads, head_dim, page_size);
        LLM_CHECK_LAUNCH("kv4_read");
        return 0;
    });
}

LLM_TRACE_EXPORT(kv4_store)
