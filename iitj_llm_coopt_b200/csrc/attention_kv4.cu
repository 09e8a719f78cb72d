// Attention over the packed key/value cache (format: kv4.cuh): the general kernel.
//
// Any head size (a multiple of 32 up to 256), any page size (a multiple of 4), both engine types, any mix of prompt portions and
// single tokens: one block a token row and key/value head, for up to four of the group's query heads at a time.  Every number of the
// cache is taken apart once per block, as z + s n in float32, and enters float32 products.
//
//   scores   a lane is a key: it reads its key's words and adds q . k for the block's query heads, q broadcast from shared memory
//   softmax  running maximum and sum a head and warp (a block's warps take the 32-key chunks in turn, so they see different keys)
//   values   a lane is four numbers of the value head (a half-word of codes), the chunk's probabilities broadcast from shared memory
// and at the end the warps' sums are joined.  Keys outside [lo, pos] are not read.
//
// What bounds it is latency, of about 1700 instructions and the value rows' loads a chunk and warp; so the keys of few rows are split
// over blocks, whose sums a second kernel joins.  Single tokens in float32: five contexts of 300 to 900 keys, 32 / 8 heads of 64, 18.4 us
// (without splits, by blocks of sixteen warps: 40.6; with half the lanes idle over heads of 64 numbers: 24.0); one of 32000 keys, 32 / 8
// heads of 128, 81 us; eight of 8192 113 us.  Other head sizes in bfloat16, 32 / 8 heads: eight contexts of 8192 keys 121 (32 numbers a
// head), 184 (96) and 350 us (256), a prompt of 512 tokens, a block a row, 229, 279 and 531 us.
// Sums are of p v with the largest p 1, in float32: they leave its range where the sum of a row's p |v| does, as the unpacked kernels' do.
#include "kv4.cuh"

namespace {

constexpr int kGenHeads = 4, kGenWarps = 4;

template <typename T> __device__ __forceinline__ T of_float(float v) { return from_f32<T>(v); }

// The keys of a row that a split takes, and how many splits there are work for: from the row's own context, so that a captured graph
// follows it as it grows.
struct GenSpan { int per, splits; };
__device__ __forceinline__ GenSpan gen_span(int pos, int lo, int splits) {
    const int keys = pos - lo + 1, per = ((keys + splits - 1) / splits + 31) & ~31;
    return {per, (keys + per - 1) / per};
}

// Weight of a sum relative to m among sums of which the largest m is `top`.  (m is -inf where no key was seen, or only keys of NaN.)
__device__ __forceinline__ float gen_weight(float m, float l, float top) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - top); }

// GT: groups of a head as a constant (a key's words then come in a few wide loads, all asked for at once), or 0.
template <typename T, int GT>
__global__ void __launch_bounds__(32 * kGenWarps)
attn_kv4_general_kernel(const T* __restrict__ q, int q_stride, const uint8_t* __restrict__ cache, const int* __restrict__ block_table,
                        int table_width, const int* __restrict__ rows, const int* __restrict__ token_request, const int* __restrict__ positions, T* __restrict__ out,
                        int out_stride, int heads, int kv_heads, int head_dim, int page_size, int window, float sl, int splits, float* part) {
    pdl_trigger();
    pdl_wait();
    __shared__ __align__(16) float sq[kGenHeads][kKv4MaxDim];
    __shared__ float sp[kGenWarps][kGenHeads][32];
    __shared__ float sm[kGenWarps][kGenHeads], sl_sum[kGenWarps][kGenHeads];
    const int t = rows ? rows[blockIdx.x] : blockIdx.x, hk = blockIdx.y, D = GT ? 32 * GT : head_dim, G = GT ? GT : D / 32, group = heads / kv_heads;
    const int ht = blockIdx.z / splits, split = blockIdx.z - ht * splits, h0 = hk * group + ht * kGenHeads, nh = min(kGenHeads, group - ht * kGenHeads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pos = positions[t], lo = window > 0 ? max(0, pos - window + 1) : 0;
    const GenSpan span = gen_span(pos, lo, splits);
    if (split >= span.splits) return;
    const int first = lo + split * span.per, last = min(pos, first + span.per - 1);
    const int* table = block_table + (size_t)token_request[t] * table_width;
    const size_t block_bytes = kv4_block_bytes(page_size, G);
    for (int i = threadIdx.x; i < kGenHeads * D; i += (32 * kGenWarps)) {
        const int h = i / D, c = i - h * D;
        sq[h][c] = h < nh ? to_f32(q[(size_t)t * q_stride + (size_t)(h0 + h) * D + c]) * sl : 0.f;       // (scores in log2 units)
    }
    __syncthreads();
    // this lane's value numbers: half-words lane and lane + 32 of a row; of 64 numbers, half-word lane % 16 of every other row
    constexpr int kRows = GT == 2 ? 2 : 1, kUnits = GT ? 1 : 2;
    const int units = 8 * G, unit = lane & (32 / kRows - 1);
    float o[kUnits][kGenHeads][4], m[kGenHeads], l[kGenHeads];
#pragma unroll
    for (int h = 0; h < kGenHeads; ++h) {
        m[h] = -INFINITY; l[h] = 0.f;
#pragma unroll
        for (int r = 0; r < kUnits; ++r) o[r][h][0] = o[r][h][1] = o[r][h][2] = o[r][h][3] = 0.f;
    }
    for (int k0 = first + warp * 32; k0 <= last; k0 += kGenWarps * 32) {
        const int n = min(32, last + 1 - k0), key = k0 + min(lane, n - 1);
        const int lp = key / page_size, off = key - lp * page_size, page = table[lp];
        const uint8_t* block = cache + ((size_t)page * kv_heads + hk) * block_bytes;
        const uint32_t* codes = reinterpret_cast<const uint32_t*>(block + (size_t)off * 16 * G);
        const uint32_t* par = reinterpret_cast<const uint32_t*>(block + kv4_key_par(page_size, G) + (size_t)off * 4 * G);
        float s[kGenHeads];
#pragma unroll
        for (int h = 0; h < kGenHeads; ++h) s[h] = 0.f;
        auto add_word = [&](uint32_t w, uint32_t p, int g, int j) {
            const float step = kv4_step(p), zero = kv4_zero(p);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = fmaf(step, (float)((w >> kv4_bit(e)) & 15u), zero);
#pragma unroll
            for (int h = 0; h < kGenHeads; ++h) {
                const float4 a = *reinterpret_cast<const float4*>(&sq[h][32 * g + 8 * j]), b = *reinterpret_cast<const float4*>(&sq[h][32 * g + 8 * j + 4]);
                s[h] += ((a.x * x[0] + a.y * x[1]) + (a.z * x[2] + a.w * x[3])) + ((b.x * x[4] + b.y * x[5]) + (b.z * x[6] + b.w * x[7]));
            }
        };
        if constexpr (GT > 0) {
            struct alignas(4 * GT) Words { uint32_t w[GT]; };
            const Words p = *reinterpret_cast<const Words*>(par);
            Words c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = reinterpret_cast<const Words*>(codes)[j];
#pragma unroll
            for (int g = 0; g < GT; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) add_word(c[j].w[g], p.w[g], g, j);
        } else {
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) add_word(codes[j * G + g], par[g], g, j);
        }
        __syncwarp();                                    // the chunk before is done with sp
#pragma unroll
        for (int h = 0; h < kGenHeads; ++h) {
            const float v = lane < n ? s[h] : -INFINITY;
            const float top = fmaxf(m[h], warp_max(v));
            const float mu = top == -INFINITY ? 0.f : top;              // (every score -inf so far: nothing to be relative to)
            const float f = exp2f(m[h] - mu), p = lane < n ? exp2f(v - mu) : 0.f;
            m[h] = top;
            l[h] = l[h] * f + p;
#pragma unroll
            for (int r = 0; r < kUnits; ++r) { o[r][h][0] *= f; o[r][h][1] *= f; o[r][h][2] *= f; o[r][h][3] *= f; }
            sp[warp][h][lane] = p;
        }
        __syncwarp();
#pragma unroll 4
        for (int i = 0; i < n; i += kRows) {
            const int at = i + (kRows > 1 ? lane / 16 : 0), row = min(at, n - 1);        // (behind the last key: it again, times 0)
            const int voff = __shfl_sync(0xffffffffu, off, row);
            const uint8_t* vb = cache + ((size_t)__shfl_sync(0xffffffffu, page, row) * kv_heads + hk) * block_bytes;
            const uint16_t* vc = reinterpret_cast<const uint16_t*>(vb + kv4_value_codes(page_size, G) + (size_t)voff * 16 * G);
            const uint32_t* vpar = reinterpret_cast<const uint32_t*>(vb + kv4_value_par(page_size, G) + (size_t)voff * 4 * G);
#pragma unroll
            for (int r = 0; r < kUnits; ++r) {
                const int u = unit + 32 * r;
                if (GT || u < units) {
                    const uint32_t w = vc[u], p4 = vpar[u % G];
                    const float step = kv4_step(p4), zero = kv4_zero(p4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = fmaf(step, (float)((w >> (4 * e)) & 15u), zero);
#pragma unroll
                        for (int h = 0; h < kGenHeads; ++h) o[r][h][e] = fmaf(sp[warp][h][at], x, o[r][h][e]);
                    }
                }
            }
        }
    }
    if constexpr (kRows > 1) {
#pragma unroll
        for (int h = 0; h < kGenHeads; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[0][h][e] += __shfl_xor_sync(0xffffffffu, o[0][h][e], 16);
    }
    auto top_of = [&](int h) {
        float top = sm[0][h];
        for (int w = 1; w < kGenWarps; ++w) top = fmaxf(top, sm[w][h]);
        return top;
    };
#pragma unroll
    for (int h = 0; h < kGenHeads; ++h) {
        l[h] = warp_sum(l[h]);
        if (lane == 0) { sm[warp][h] = m[h]; sl_sum[warp][h] = l[h]; }
    }
    __syncthreads();
    // joined over the warps, one after another, into the query rows' place
    for (int w = 0; w < kGenWarps; ++w) {
        if (warp == w) {
            for (int h = 0; h < nh; ++h) {
                const float top = top_of(h);
                const float f = gen_weight(sm[w][h], sl_sum[w][h], top);
#pragma unroll
                for (int r = 0; r < kUnits; ++r) {
                    const int u = lane + 32 * r;
                    if (u < units) {
                        const int c = u / G, g = u - c * G, at = 32 * g + 8 * (c >> 1) + (c & 1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = 0.f;
                            // (a loop over h with o[r][h] in registers: selected by comparison)
#pragma unroll
                            for (int hh = 0; hh < kGenHeads; ++hh) if (hh == h) v = o[r][hh][e];
                            sq[h][at + 2 * e] = (w == 0 ? 0.f : sq[h][at + 2 * e]) + f * v;
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < nh * D; i += (32 * kGenWarps)) {
        const int h = i / D, c = i - h * D;
        const float top = top_of(h);
        float sum = 0.f;
        for (int w = 0; w < kGenWarps; ++w) sum += sl_sum[w][h] * gen_weight(sm[w][h], sl_sum[w][h], top);
        if (span.splits == 1) {
            out[(size_t)t * out_stride + (size_t)(h0 + h) * D + c] = of_float<T>(sq[h][c] / sum);
        } else {
            float* to = part + (((size_t)blockIdx.x * heads + h0 + h) * splits + split) * (D + 2);
            to[2 + c] = sq[h][c];
            if (c == 0) { to[0] = top; to[1] = sum; }
        }
    }
}

// Joins the splits of a row and head, a warp each.  part: [rows][heads][splits][2 + head_dim] (reference, sum, numbers)
template <typename T>
__global__ void __launch_bounds__(128)
attn_kv4_general_join_kernel(const float* __restrict__ part, const int* __restrict__ rows, const int* __restrict__ positions, T* __restrict__ out,
                             int out_stride, int heads, int D, int window, int splits) {
    pdl_trigger();
    pdl_wait();
    const int head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= heads) return;
    const int t = rows ? rows[blockIdx.x] : blockIdx.x, pos = positions[t];
    const int n = gen_span(pos, window > 0 ? max(0, pos - window + 1) : 0, splits).splits;
    if (n == 1) return;                                  // one block wrote the result itself
    const float* from = part + ((size_t)blockIdx.x * heads + head) * splits * (D + 2);
    float top = -INFINITY;
    for (int s = 0; s < n; ++s) top = fmaxf(top, from[(size_t)s * (D + 2)]);
    float sum = 0.f, v[kKv4MaxDim / 32];
#pragma unroll
    for (int e = 0; e < kKv4MaxDim / 32; ++e) v[e] = 0.f;
#pragma unroll 2
    for (int s = 0; s < n; ++s) {
        const float* p = from + (size_t)s * (D + 2);
        const float f = gen_weight(p[0], p[1], top);
        sum += f * p[1];
#pragma unroll
        for (int e = 0; e < kKv4MaxDim / 32; ++e)
            if (32 * e < D) v[e] += f * p[2 + 32 * e + lane];
    }
#pragma unroll
    for (int e = 0; e < kKv4MaxDim / 32; ++e)
        if (32 * e < D) out[(size_t)t * out_stride + (size_t)head * D + 32 * e + lane] = of_float<T>(v[e] / sum);
}

}  // namespace

// part: [n_rows][heads][splits][2 + head_dim] where splits is above 1.
// rows: [n_rows] the token rows to work on, null: rows 0 .. n_rows - 1.  q: [tokens, q_stride], head h at columns [h * head_dim, ...); cache: pages of kv_heads blocks (kv4.cuh).
LLM_API int llm_attention_kv4_general(const void* q, int q_stride, const void* cache, const int* block_table, int table_width,
                                      const int* rows, int n_rows, const int* token_request, const int* positions, void* out, int out_stride, int dtype, int heads,
                                      int kv_heads, int head_dim, int page_size, int window, float scale, int splits, float* part, cudaStream_t stream) {
    if (n_rows == 0) return 0;
    if (!kv4_geometry(head_dim, page_size) || kv_heads <= 0 || heads % kv_heads)
        LLM_FAIL(-1, "attention_kv4: heads %d / kv_heads %d / head_dim %d / page %d not supported", heads, kv_heads, head_dim, page_size);
    const int tiles = (heads / kv_heads + kGenHeads - 1) / kGenHeads;
    if (splits < 1 || (splits > 1 && !part)) LLM_FAIL(-1, "attention_kv4: %d splits%s", splits, splits > 1 ? " without a place for their sums" : "");
    if (kv_heads > 65535 || (long long)tiles * splits > 65535) LLM_FAIL(-1, "attention_kv4: too many heads or splits");
    return llm_dispatch_dtype(dtype, [&](auto tag) {
        using T = decltype(tag);
        auto go = [&](auto kernel) {
            llm_launch(kernel, dim3(n_rows, kv_heads, tiles * splits), 32 * kGenWarps, 0, stream, (const T*)q, q_stride, (const uint8_t*)cache,
                       block_table, table_width, rows, token_request, positions, (T*)out, out_stride, heads, kv_heads, head_dim, page_size, window,
                       scale * 1.4426950408889634f, splits, part);
        };
        if (head_dim == 64) go(attn_kv4_general_kernel<T, 2>);
        else if (head_dim == 128) go(attn_kv4_general_kernel<T, 4>);
        else go(attn_kv4_general_kernel<T, 0>);
        if (splits > 1)
            llm_launch(attn_kv4_general_join_kernel<T>, dim3(n_rows, (heads + 3) / 4), 128, 0, stream, (const float*)part, rows, positions, (T*)out,
                       out_stride, heads, head_dim, window, splits);
        LLM_CHECK_LAUNCH("attention_kv4");
        return 0;
    });
}

LLM_TRACE_EXPORT(attention_kv4)
