// Attention of single tokens (one query token per request) over the packed key/value cache (format: kv4.cuh), bfloat16, head sizes 64
// and 128, pages whose size divides 32 or is a multiple of it.
//
// What bounds it is reading the codes: 40 G bytes a token and key/value head (160 at head size 128), each read once.  The codes are
// taken apart in registers, right into the operands of the matrix instructions, so the arithmetic beside the reading has to stay small:
// about an instruction a number and lane.
//
// A warp walks tiles of 32 keys by itself: its ring of stages in shared memory is filled by 16-byte asynchronous copies of its own lanes
// (bulk copies, eight a tile, cost their issuing lanes about 100 clocks each: 1600 of a tile's 4000); warps do not wait for one
// another until the end.  A block takes one split of an item's tiles, dealt out in turn to its warps, and joins their sums; with more
// than one split the blocks leave theirs in scratch memory, and a second kernel joins those.
//
// Measured, 32 heads over 8 of 128 numbers, over six inputs in turn: 8 requests over 8192 tokens 32.4 us, 2.6 TB/s of codes (the reading
// alone would take 12.8); 2 over 32000 tokens 32.9; one over 4096 tokens 12.6, over 32000 25.4.  8 over 8192 of 64 numbers a head: 22.1.
// What bounds it is not one thing.  Of 8 x 8192 a capture says: 950 instructions a tile of 32 keys and 8 heads with all that is around the
// loop, which fill 51% of the issue slots of an SM while it works (ALU pipe 43%, tensor pipe 16%); 2.6 warps a scheduler, which wait for
// what they need next rather than for a slot (stalls an issue: fixed latencies 0.89, loads 0.81, the pipes 0.49, shared memory 0.32); and a
// fifth of the time in which an SM has nothing to do (256 blocks on 296 places: 40 SMs have one where the others have two).
//
//   scores   mma m16n8k16, 16 keys x 8 query heads.  A code n becomes the float16 1024 + n or 64 + n by one AND-OR (its last mantissa
//            bits count 1 or 1/16), an exact number; q is float16 too, exactly, behind a power of two.  Per group of 32 the products' sum S
//            over those gives the score's part as s S + z sum q - s sum (1024 or 64) q.  The last two terms of all groups are two more
//            products: one operand are the stored (s, z) words as they lie, the other one the sums of q (as three bfloat16 each).  Nothing
//            of the key is rounded.
//   values   the transposed product, 16 numbers x 8 heads over 16 keys: the operand is n - 8 (128 + n - 136, exact), the other one
//            p s, rounded once to bfloat16 (float16 would not hold s), a group at a time.  p crosses the lanes as float16, times 2^7 so that
//            what is flushed lies 2^-32 below a row's largest.  The middles z + 8 s (rounded to bfloat16: they are small beside the
//            numbers) and the sum of p are one more product, of rows of middles and of ones, with p as bfloat16.
//            (About the zero points, with n for n - 8, the two parts nearly cancel over a long context: at 32000 keys the result was 5.2e-3
//            off the one in 64 bits; it is 2.3e-3, of which bfloat16's last rounding alone makes 1.7e-3.  p and p s each rounded to
//            bfloat16: 2.7e-3, and 30.8 us instead of 31.8.  Over contexts of 500 to 32000 tokens the result is 2.1e-3 to 2.4e-3 off: p s and
//            the middles' p are each rounded by themselves, and the sum is of the latter.)
//   range    p is up to 2^15 here, so p s would leave float32 and bfloat16 from steps of 2^113 on, and so would the products' 2^17 times a
//            key's step.  From the first tile with a value's step or zero point of 2^65 or more a warp's sums are taken times 2^-64
//            (its reference counts that); a tile with such a key has its stored words multiplied by 2^-64 where they lie in shared memory
//            and its scores made again, with a scale times 2^64.  The vote on the reference
//            finds out; looking at the words costs 3% (8 requests over 8192: 31.5 to 32.5 us).
// The order of codes in a row (kv4.cuh) is the order in which these instructions' lanes want them: no shuffle, one 4 G-byte load of a
// key row and one 2 G-byte load of a value row per lane.
#include "kv4.cuh"

#include <cuda_fp16.h>

namespace {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

constexpr int kTile = 32;               // keys of a warp's step
// Six warps a block and two blocks an SM leave a thread 168 registers, which the two chains of the loop need (eight warps with 128:
// 8 x 8192 keys at 32 / 8 heads of 128 in 33.5 us instead of 29.8; blocks of four, three an SM: 30.2 us, and 37 uneven contexts of 600
// keys 17.4 us instead of 13.7; all before p s was rounded only once and before the words were looked at).
constexpr int kWarps = 6, kResident = 2;
constexpr float kStep = 8.f, kLift = 7.f;       // (log2 units) a reference's lag at most; p's factor
constexpr int kHeads = 8;               // query heads of a block (columns of the products)
template <int G> __host__ __device__ constexpr int stages() { return G == 4 ? 3 : 4; }
template <int G> __host__ __device__ constexpr int stage_bytes() { return kTile * kKv4TokenBytes * G; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// BYTES of global memory to shared memory, asynchronously; zeros in their place where `take` is false (nothing is read then).
template <int BYTES> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool take) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(take ? BYTES : 0), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a . b of float16 operands.
__device__ __forceinline__ void mma16816_half_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma16816_half(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 halves_of(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// (w & MASK) | base in one instruction (the compiler makes two of the expression).
template <uint32_t MASK> __device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t base) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w), "n"(MASK), "r"(base));
    return x;
}
// Two codes (bits 0-3 and 16-19 of w) as the float16 numbers 1024 + n; two codes of bits 4-7 and 20-23 as 64 + n.
__device__ __forceinline__ uint32_t half_codes_low(uint32_t w) { return and_or<0x000f000fu>(w, 0x64006400u); }
__device__ __forceinline__ uint32_t half_codes_high(uint32_t w) { return and_or<0x00f000f0u>(w, 0x54005400u); }
// Two codes (bits 0-3 and 16-19 of w) as the bfloat16 numbers n - 8: 128 + n - 136.
__device__ __forceinline__ uint32_t codes(uint32_t w) {
    const uint32_t x = and_or<0x000f000fu>(w, 0x43004300u);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(136.f));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// z + 8 s of two tokens' (s, z) words.
__device__ __forceinline__ uint32_t middles(uint32_t a, uint32_t b) {
    const uint32_t s = __byte_perm(a, b, 0x5410), z = __byte_perm(a, b, 0x7632);
    const __nv_bfloat162 m = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&s), __float2bfloat162_rn(8.f), *reinterpret_cast<const __nv_bfloat162*>(&z));
    return *reinterpret_cast<const uint32_t*>(&m);
}

template <int G> struct alignas(4 * G) Words { uint32_t w[G]; };

// (s, z) words of a token in which a number is 2^65 or more in size (both top bits of its exponent are set), or NaN.
template <int G> __device__ __forceinline__ uint32_t loud(const Words<G>& x) {
    uint32_t both = 0u;
#pragma unroll
    for (int g = 0; g < G; ++g) both |= x.w[g] & (x.w[g] << 1);
    return both & 0x40004000u;
}
constexpr float kQuiet = 5.42101086242752217e-20f, kLoud = 18446744073709551616.f;      // 2^-64 and 2^64
constexpr float kLoudLog = 64.f;
template <int G> struct alignas(2 * G) Halves { uint32_t w[G / 2]; };      // G half-words of a value row
template <typename W> __device__ __forceinline__ W lds(const unsigned char* at) { return *reinterpret_cast<const W*>(at); }

struct SingleArgs {
    const bf16* q;
    int q_stride;
    const uint8_t* cache;
    const int* block_table;
    int table_width;
    const int* items;               // token rows
    const int* token_request;
    const int* positions;
    bf16* out;
    int out_stride;
    int heads, kv_heads, page_size, head_tiles, window;
    int split_tiles, max_splits;    // tiles of 32 keys a block takes; the splits that the launch provides for an item
    float* part_o;                  // [items][heads][max_splits][D], relative to the split's reference
    float* part_ml;                 // [items][heads][max_splits][2]: reference (log2 units; -inf: no sum), sum
    float sl;                       // softmax scale * log2(e)
};

// The tiles of an item at `pos`, and how many of them a split takes: split_tiles, or more where the launch provides too few splits (a
// captured graph's contexts grow).
struct Span { int first, tiles, per_split, splits; };
__device__ __forceinline__ Span span_of(const SingleArgs& a, int pos) {
    Span s;
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    s.first = lo / kTile;
    s.tiles = pos / kTile - s.first + 1;
    s.per_split = max(a.split_tiles, (s.tiles + a.max_splits - 1) / a.max_splits);
    s.splits = (s.tiles + s.per_split - 1) / s.per_split;
    return s;
}

// grid (max_splits, kv_heads * head_tiles, items)
template <int G>
__global__ void __launch_bounds__(kWarps * 32, kResident)
attn_kv4_single_kernel(const SingleArgs a) {
    pdl_trigger();
    constexpr int D = 32 * G, kStages = stages<G>(), kStageBytes = stage_bytes<G>();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float sm_m[kWarps][kHeads], sm_l[kWarps][kHeads];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r8 = lane >> 2, j = lane & 3;
    const int split = blockIdx.x;
    const int hk = blockIdx.y / a.head_tiles, ht = blockIdx.y - hk * a.head_tiles;
    const int group = a.heads / a.kv_heads, h0 = hk * group + ht * kHeads, nh = min(kHeads, group - ht * kHeads);
    // (No kernel of this library writes a step's index arrays, and none but its kernels lets the next one start early: the index
    // arrays are there before the wait.  Queries, keys and values come from the kernels before this one.)
    const int tok = a.items[blockIdx.z], pos = a.positions[tok];
    const int* table = a.block_table + (size_t)a.token_request[tok] * a.table_width;
    const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const Span span = span_of(a, pos);
    if (split >= span.splits) return;
    const int first = span.first + split * span.per_split + warp, last = span.first + min(span.tiles, (split + 1) * span.per_split) - 1;
    constexpr int stride = kWarps;                       // this warp's tiles: first, first + stride, ... up to last
    const int n_tiles = first <= last ? (last - first) / stride + 1 : 0;
    // A stage is laid out as a page of 32 tokens is.  Lane x copies the parameters of token x, and 16 bytes of the codes of the tokens
    // x / G, x / G + 32 / G, ...  (A page's tokens divide a tile's 32, or a tile lies in one page.)
    constexpr int kRowStep = kTile / G;
    const int ps = a.page_size, page_shift = ps <= kTile ? 31 - __clz(ps) : 5, row_mask = min(ps, kTile) - 1;
    const size_t block_bytes = kv4_block_bytes(ps, G), page_bytes = (size_t)a.kv_heads * block_bytes;
    const uint8_t* cache = a.cache + (size_t)hk * block_bytes;
    const int key_par = kv4_key_par(ps, G) + (lane & row_mask) * 4 * G, value_par = key_par + ps * 20 * G;
    const int code_at = (lane / G & row_mask) * 16 * G + (lane % G) * 16, value_codes = ps * 20 * G;
    unsigned char* ring = smem + warp * kStages * kStageBytes;
    const uint32_t ring_at = smem_u32(ring), par_to = kTile * 16 * G + lane * 4 * G, code_to = lane * 16;
    // The page of token `lane` of a tile, asked for a tile's time before it is used (a key behind the token: the token's page; one
    // before the window: the window's first).
    auto fetch_page = [&](int i) {
        if (i >= n_tiles) return 0;
        const int key0 = (first + i * stride) * kTile, key = max(min(key0 + lane, pos), lo);
        return table[ps <= kTile ? key >> page_shift : key0 / ps];
    };
    auto load_tile = [&](int i, int page) {              // all lanes; tile number i of this warp
        if (i < n_tiles) {
            const int key0 = (first + i * stride) * kTile, skip = ps <= kTile ? 0 : key0 % ps;       // tokens of the page before the tile
            const uint32_t dst = ring_at + (i % kStages) * kStageBytes;
            const bool inside = key0 + kTile - 1 <= pos && key0 >= lo;
            const bool take = inside || (key0 + lane <= pos && key0 + lane >= lo);
            const uint8_t* block = cache + (size_t)page * page_bytes + skip * 4 * G;
            copy_async<4 * G>(dst + par_to, block + key_par, take);
            copy_async<4 * G>(dst + par_to + kTile * 20 * G, block + value_par, take);
#pragma unroll
            for (int x = 0; x < G; ++x) {
                const int row = x * kRowStep + lane / G;
                const bool take_row = inside || (key0 + row <= pos && key0 + row >= lo);
                const uint8_t* codes = cache + (size_t)__shfl_sync(0xffffffffu, page, row) * page_bytes + skip * 16 * G + ((x * kRowStep & row_mask) * 16 * G + code_at);
                copy_async<16>(dst + x * kRowStep * 16 * G + code_to, codes, take_row);
                copy_async<16>(dst + kTile * 20 * G + x * kRowStep * 16 * G + code_to, codes + value_codes, take_row);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int pages[kStages], page_next = 0;
#pragma unroll
    for (int i = 0; i < kStages; ++i) pages[i] = fetch_page(i);
    page_next = fetch_page(kStages);
    pdl_wait();
#pragma unroll
    for (int i = 0; i < kStages; ++i) load_tile(i, pages[i]);

    // Queries: column r8 of the product is head h0 + r8; the lane holds numbers 32 g + 8 j .. + 7 of it.
    // They become float16 (which holds a bfloat16's eight bits) after a division by a power of two, the largest number's; what that
    // pushes below float16's range is 2^-24 of the largest.
    uint32_t qb[G][4], qz[3] = {0u, 0u, 0u};
    float slh[2];                    // the scale of this lane's two columns, that power of two in it
    {
        uint4 raw[G];
        uint32_t top = 0u;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            raw[g] = make_uint4(0u, 0u, 0u, 0u);
            if (r8 < nh) raw[g] = *reinterpret_cast<const uint4*>(a.q + (size_t)tok * a.q_stride + (size_t)(h0 + r8) * D + 32 * g + 8 * j);
            const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e8 = min(max((int)(top >> 23), 1), 253);                       // (biased exponent; NaN and infinity stay what they are)
        const float down = __uint_as_float((uint32_t)(254 - e8) << 23), up = __uint_as_float((uint32_t)e8 << 23) * a.sl;
        slh[0] = __shfl_sync(0xffffffffu, up, 8 * j);
        slh[1] = __shfl_sync(0xffffffffu, up, 8 * j + 4);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const uint32_t w[4] = {raw[g].x, raw[g].y, raw[g].z, raw[g].w};
            float sum = 0.f, shifted = 0.f;                                      // sum of q, and of q times what its codes have on top
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = __uint_as_float(w[e] << 16) * down, y = __uint_as_float(w[e] & 0xffff0000u) * down;
                const __half2 h = __floats2half2_rn(x, y);
                qb[g][e] = *reinterpret_cast<const uint32_t*>(&h);
                const float xy = __low2float(h) + __high2float(h);
                sum += xy;
                shifted += (e & 1 ? 64.f : 1024.f) * xy;
            }
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                sum += __shfl_xor_sync(0xffffffffu, sum, d);
                shifted += __shfl_xor_sync(0xffffffffu, shifted, d);
            }
            // the operands that meet (s, z) of group j, in three bfloat16 each
            if (j == g) {
                float neg = -shifted;
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    const float hn = __bfloat162float(__float2bfloat16_rn(neg)), hs = __bfloat162float(__float2bfloat16_rn(sum));
                    qz[e] = pack_pair(hn, hs);
                    neg -= hn;
                    sum -= hs;
                }
            }
        }
    }
    float o[G][2][4], oz[4] = {0.f, 0.f, 0.f, 0.f}, m[2] = {0.f, 0.f};
    float quiet = 1.f;               // 2^-64 once a value of this warp was loud: in all its sums
    bool has[2] = {false, false};    // m holds a reference (in log2 units)
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[g][e][0] = o[g][e][1] = o[g][e][2] = o[g][e][3] = 0.f;
    // Row x of a 16-row product is token (x / 2) + 4 (x % 2) of its eight, so that the four lanes of a value load read four
    // neighbouring tokens.
    const int trow = (r8 >> 1) + 4 * (r8 & 1);
    constexpr int kKeyPar = kTile * 16 * G, kValue = kTile * 20 * G, kValuePar = kTile * 36 * G;
    const int key_at = trow * 16 * G + 4 * G * j, par_at = trow * 4 * G, value_at = kValue + j * 16 * G + 2 * G * r8;
    const int kz_at = kKeyPar + par_at + 4 * (G == 4 ? j : j & 1), vz_at = kValuePar + j * 4 * G + 4 * (r8 < G ? r8 : 0);
    const uint32_t z_keep = r8 < G ? 0xffffffffu : 0u, z_add = r8 == G ? 0x3f803f80u : 0u;         // rows of oz: z of the groups, then 1

    // Whether token x of a tile (lane x) has loud numbers in its key or its value.
    auto loud_key = [&](const unsigned char* base) { return loud<G>(lds<Words<G>>(base + kKeyPar + lane * 4 * G)); };
    auto loud_value = [&](const unsigned char* base) { return loud<G>(lds<Words<G>>(base + kValuePar + lane * 4 * G)); };
    auto scores = [&](const unsigned char* base, float (&sc)[2][4]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned char* ku = base + 16 * u * 16 * G;
            const unsigned char* pu = base + 16 * u * 4 * G;
            const Words<G> k0 = lds<Words<G>>(ku + key_at), k1 = lds<Words<G>>(ku + key_at + 8 * 16 * G);
            const Words<G> p0 = lds<Words<G>>(pu + kKeyPar + par_at), p1 = lds<Words<G>>(pu + kKeyPar + par_at + 8 * 4 * G);
            uint32_t z0 = lds<uint32_t>(pu + kz_at), z1 = lds<uint32_t>(pu + kz_at + 8 * 4 * G);
            if (G < 4 && j >= G) z0 = z1 = 0u;
            sc[u][0] = sc[u][1] = sc[u][2] = sc[u][3] = 0.f;
            mma16816(sc[u], z0, z1, z0, z1, qz[0], qz[1]);               // sum over the groups of z sum q - s sum (1024 or 64) q
            mma16816(sc[u], z0, z1, 0u, 0u, qz[2], 0u);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float c[4];
                const uint32_t x = k0.w[g], y = k1.w[g];
                const uint32_t xs = x >> 8, ys = y >> 8;
                mma16816_half_first(c, half_codes_low(x), half_codes_low(y), half_codes_high(x), half_codes_high(y), qb[g][0], qb[g][1]);
                mma16816_half(c, half_codes_low(xs), half_codes_low(ys), half_codes_high(xs), half_codes_high(ys), qb[g][2], qb[g][3]);
                const float s0 = kv4_step(p0.w[g]), s1 = kv4_step(p1.w[g]);
                sc[u][0] = fmaf(s0, c[0], sc[u][0]);
                sc[u][1] = fmaf(s0, c[1], sc[u][1]);
                sc[u][2] = fmaf(s1, c[2], sc[u][2]);
                sc[u][3] = fmaf(s1, c[3], sc[u][3]);
            }
        }
    };
    // Exponents t of a tile relative to the reference m.  It follows the maximum in steps of 2^8 only (p stays below 2^8), so that in
    // most tiles one vote is all there is to do; a head without a reference yet takes the tile's maximum.
    auto exponents = [&](int i, unsigned char* base, uint32_t odd, float (&sc)[2][4], float (&t)[2][4]) {
        const int key0 = (first + i * stride) * kTile;
        float sl[2] = {slh[0], slh[1]};
        auto mask = [&] {
            if (key0 + kTile - 1 > pos || key0 < lo) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = key0 + 16 * u + 8 * e + trow;
                        if (key > pos || key < lo) sc[u][2 * e] = sc[u][2 * e + 1] = -INFINITY;
                    }
            }
        };
        auto relative = [&] {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[u][e] = fmaf(sc[u][e], sl[e & 1], -m[e & 1]);
        };
        mask();
        relative();
        const float over = fmaxf(max3(max3(t[0][0], t[0][1], t[0][2]), t[0][3], t[1][0]), max3(t[1][1], t[1][2], t[1][3]));
        if (__any_sync(0xffffffffu, !has[0] || !has[1] || over > kStep + kLift || odd != 0u)) {
            if (__any_sync(0xffffffffu, odd != 0u)) {
                if (__any_sync(0xffffffffu, loud_key(base) != 0u)) {     // the scores once more, over words times 2^-64
                    Words<G>* key = reinterpret_cast<Words<G>*>(base + kKeyPar + lane * 4 * G);
#pragma unroll
                    for (int g = 0; g < G; ++g) key->w[g] = pack_pair(kv4_step(key->w[g]) * kQuiet, kv4_zero(key->w[g]) * kQuiet);
                    __syncwarp();
                    scores(base, sc);
                    mask();
                    sl[0] *= kLoud;
                    sl[1] *= kLoud;
                }
                if (quiet == 1.f && __any_sync(0xffffffffu, loud_value(base) != 0u)) {
                    quiet = kQuiet;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        oz[e] *= kQuiet;
#pragma unroll
                        for (int g = 0; g < G; ++g) { o[g][0][e] *= kQuiet; o[g][1][e] *= kQuiet; }
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = fmaxf(fmaxf(sc[0][e], sc[0][2 + e]), fmaxf(sc[1][e], sc[1][2 + e])) * sl[e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float now = (has[e] ? fmaxf(m[e] + kLift, top) : top) - kLift;
                const float f = has[e] ? ex2(m[e] - now) : 0.f;          // (the sums are 0, or NaN, before the first reference)
                has[e] = now > -INFINITY;                                // (no key yet, or keys of NaN: any reference will do)
                m[e] = has[e] ? now : 0.f;
                oz[e] *= f;
#pragma unroll
                for (int g = 0; g < G; ++g) { o[g][0][e] *= f; o[g][0][2 + e] *= f; o[g][1][e] *= f; o[g][1][2 + e] *= f; }
            }
            relative();
        }
    };
    auto values = [&](const unsigned char* base, const float (&t)[2][4]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float2 f0 = halves_of(transposed8x8(half_pair(ex2(t[u][0]), ex2(t[u][1]))));
            float2 f1 = halves_of(transposed8x8(half_pair(ex2(t[u][2]), ex2(t[u][3]))));
            f0.x *= quiet; f0.y *= quiet; f1.x *= quiet; f1.y *= quiet;
            const uint32_t p0 = pack_pair(f0.x, f0.y), p1 = pack_pair(f1.x, f1.y);
            const unsigned char* vu = base + 16 * u * 16 * G;
            const unsigned char* pu = base + 16 * u * 4 * G;
            {   // rows of the groups' middles, and a row of ones, over the 16 tokens, times p
                const uint32_t wa = lds<uint32_t>(pu + vz_at), wb = lds<uint32_t>(pu + vz_at + 4 * 4 * G);
                const uint32_t wc = lds<uint32_t>(pu + vz_at + 8 * 4 * G), wd = lds<uint32_t>(pu + vz_at + 12 * 4 * G);
                mma16816(oz, (middles(wa, wb) & z_keep) | z_add, 0u, (middles(wc, wd) & z_keep) | z_add, 0u, p0, p1);
            }
            const unsigned char* wu = pu + kValuePar + j * 4 * G;
            const Words<G> wa = lds<Words<G>>(wu), wb = lds<Words<G>>(wu + 4 * 4 * G), wc = lds<Words<G>>(wu + 8 * 4 * G), wd = lds<Words<G>>(wu + 12 * 4 * G);
            const Halves<G> va = lds<Halves<G>>(vu + value_at), vb = lds<Halves<G>>(vu + value_at + 4 * 16 * G);
            const Halves<G> vc = lds<Halves<G>>(vu + value_at + 8 * 16 * G), vd = lds<Halves<G>>(vu + value_at + 12 * 16 * G);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t b0 = pack_pair(f0.x * kv4_step(wa.w[g]), f0.y * kv4_step(wb.w[g]));
                const uint32_t b1 = pack_pair(f1.x * kv4_step(wc.w[g]), f1.y * kv4_step(wd.w[g]));
                const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
                const uint32_t ab = __byte_perm(va.w[g / 2], vb.w[g / 2], sel), cd = __byte_perm(vc.w[g / 2], vd.w[g / 2], sel);
                mma16816(o[g][0], codes(ab), codes(ab >> 4), codes(cd), codes(cd >> 4), b0, b1);
                mma16816(o[g][1], codes(ab >> 8), codes(ab >> 12), codes(cd >> 8), codes(cd >> 12), b0, b1);
            }
        }
    };

    // A tile's values are worked on beside the next tile's scores: two chains of instructions that do not wait for one another.
    if (n_tiles > 0) {
        float sc[2][4], t[2][4];
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();                                    // every lane's copies of the tile are there
        unsigned char* base = ring;
        scores(base, sc);
        exponents(0, base, loud_key(base) | loud_value(base), sc, t);
        for (int i = 0; i + 1 < n_tiles; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            unsigned char* next = ring + ((i + 1) % kStages) * kStageBytes;
            scores(next, sc);
            values(base, t);
            const uint32_t odd = loud_key(next) | loud_value(next);
            __syncwarp();                                // every lane has what it wants of tile i's stage
            load_tile(i + kStages, page_next);
            page_next = fetch_page(i + kStages + 1);
            exponents(i + 1, next, odd, sc, t);
            base = next;
        }
        values(base, t);
    }

    // ---- the warps' sums joined, then the blocks' --------------------------------------------------------------------------
    // row g of oz is the middles' part of group g, row G the sum of p: this lane's columns are heads 2 j and 2 j + 1
    float zg[G][2], l[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int g = 0; g < G; ++g) zg[g][e] = __shfl_sync(0xffffffffu, oz[e], 4 * g + j);
        l[e] = __shfl_sync(0xffffffffu, oz[e], 4 * G + j);
        if (r8 == 0) { sm_m[warp][2 * j + e] = has[e] ? (quiet == 1.f ? m[e] : m[e] + kLoudLog) : -INFINITY; sm_l[warp][2 * j + e] = l[e]; }
    }
    __syncthreads();                                     // every warp is done with its stages: they become the sums' place
    float* part = reinterpret_cast<float*>(smem);        // [kWarps][kHeads][D]
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int head = 2 * j + (x & 1), c = 32 * g + 8 * (r8 >> 1) + (r8 & 1) + 4 * e + (x & 2);
                if (head < nh) part[(warp * kHeads + head) * D + c] = o[g][e][x] + zg[g][x & 1];
            }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * D; i += kWarps * 32) {
        const int h = i / D;
        float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            // (a warp without a reference has nothing, or NaN, in its sums: either counts as it is)
            const float f = sm_m[w][h] == -INFINITY ? 1.f : ex2(sm_m[w][h] - top);
            sum += f * sm_l[w][h];
            v += f * part[w * kHeads * D + i];
        }
        if (span.splits == 1) {
            a.out[(size_t)tok * a.out_stride + (size_t)h0 * D + i] = __float2bfloat16_rn(v / sum);
        } else {
            const size_t at = ((size_t)blockIdx.z * a.heads + h0 + h) * a.max_splits + split;
            a.part_o[at * D + (i - h * D)] = v;
            if (i - h * D == 0) { a.part_ml[2 * at] = top; a.part_ml[2 * at + 1] = sum; }
        }
    }
}

// Joins the splits of an item and head: a warp each, D / 32 numbers a lane.
template <int D>
__global__ void __launch_bounds__(128)
attn_kv4_single_join_kernel(const SingleArgs a) {
    pdl_trigger();
    constexpr int N = D / 32;
    const int head = blockIdx.x * 4 + (threadIdx.x >> 5), item = blockIdx.y, lane = threadIdx.x & 31;
    const int tok = a.items[item];
    const Span span = span_of(a, a.positions[tok]);
    pdl_wait();                                          // (before any way out: this grid must not end before the one it follows)
    if (head >= a.heads || span.splits == 1) return;     // (one block wrote the result itself)
    const size_t at = ((size_t)item * a.heads + head) * a.max_splits;
    float top = -INFINITY;
    for (int s = lane; s < span.splits; s += 32) top = fmaxf(top, a.part_ml[2 * (at + s)]);
    top = warp_max(top);
    float sum = 0.f, v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < span.splits; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (at + s));
        const float f = ml.x == -INFINITY ? 1.f : ex2(ml.x - top);
        sum += f * ml.y;
        const float* o = a.part_o + (at + s) * D + lane * N;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] += f * o[e];
    }
    bf16* to = a.out + (size_t)tok * a.out_stride + (size_t)head * D + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) to[e] = __float2bfloat16_rn(v[e] / sum);
}

}  // namespace

// 1 if the kernel takes this geometry.
LLM_API int llm_attention_kv4_single_supported(int heads, int kv_heads, int head_dim, int page_size) {
    return kv_heads > 0 && heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128) && page_size >= 4 &&
           (kTile % page_size == 0 || page_size % kTile == 0);
}

// Keys of a tile, warps of a block, and blocks that an SM holds at a time: what a caller plans the splits with.
LLM_API int llm_attention_kv4_single_tile() { return kTile; }
LLM_API int llm_attention_kv4_single_warps() { return kWarps; }
LLM_API int llm_attention_kv4_single_resident() { return kResident; }

// items: [n_items] token rows, one query token each.  A block takes split_tiles tiles of 32 keys; max_splits blocks are provided for an
// item and head (more keys than that covers make its blocks take more each).  part_o: n_items * heads * max_splits * head_dim floats,
// part_ml: n_items * heads * max_splits * 2 floats (unused with one split).  q rows on 16-byte boundaries.
LLM_API int llm_attention_kv4_single(const void* q, int q_stride, const void* cache, const int* block_table, int table_width, const int* items,
                                     int n_items, const int* token_request, const int* positions, float* part_o, float* part_ml, void* out,
                                     int out_stride, int heads, int kv_heads, int head_dim, int page_size, int window, float scale,
                                     int split_tiles, int max_splits, cudaStream_t stream) {
    if (n_items == 0) return 0;
    if (!llm_attention_kv4_single_supported(heads, kv_heads, head_dim, page_size))
        LLM_FAIL(-1, "attention_kv4_single: heads %d / kv_heads %d / head_dim %d / page %d not supported", heads, kv_heads, head_dim, page_size);
    if (split_tiles < 1 || max_splits < 1) LLM_FAIL(-1, "attention_kv4_single: splits of %d tiles, %d of them", split_tiles, max_splits);
    if (max_splits > 1 && (!part_o || !part_ml)) LLM_FAIL(-1, "attention_kv4_single: key splits need scratch");
    if (q_stride % 8 || ((uintptr_t)q & 15)) LLM_FAIL(-1, "attention_kv4_single: query rows must lie on 16-byte boundaries");
    SingleArgs a;
    a.q = (const bf16*)q; a.q_stride = q_stride; a.cache = (const uint8_t*)cache; a.block_table = block_table; a.table_width = table_width;
    a.items = items; a.token_request = token_request; a.positions = positions; a.out = (bf16*)out; a.out_stride = out_stride;
    a.heads = heads; a.kv_heads = kv_heads; a.page_size = page_size; a.window = window; a.sl = scale * 1.4426950408889634f;
    a.head_tiles = (heads / kv_heads + kHeads - 1) / kHeads;
    a.split_tiles = split_tiles; a.max_splits = max_splits; a.part_o = part_o; a.part_ml = part_ml;
    if ((long long)kv_heads * a.head_tiles > 65535 || n_items > 65535) LLM_FAIL(-1, "attention_kv4_single: too many heads or items");
    const dim3 grid(max_splits, kv_heads * a.head_tiles, n_items);
    auto go = [&](auto kernel, auto join, size_t smem) -> int {
        // (asked for once a device: the driver's call takes longer than the launch)
        static unsigned long long allowed[2] = {0, 0};
        int dev = 0;
        cudaGetDevice(&dev);
        unsigned long long& done = allowed[head_dim == 64];
        if (dev >= 64 || !(done >> dev & 1)) {
            LLM_ALLOW_SMEM("attention_kv4_single", kernel, smem);
            if (dev < 64) done |= 1ull << dev;
        }
        llm_launch(kernel, grid, kWarps * 32, smem, stream, a);
        LLM_CHECK_LAUNCH("attention_kv4_single");
        if (max_splits > 1) {
            llm_launch(join, dim3((heads + 3) / 4, n_items), 128, 0, stream, a);
            LLM_CHECK_LAUNCH("attention_kv4_single join");
        }
        return 0;
    };
    if (head_dim == 64) return go(attn_kv4_single_kernel<2>, attn_kv4_single_join_kernel<64>, (size_t)kWarps * stages<2>() * stage_bytes<2>());
    return go(attn_kv4_single_kernel<4>, attn_kv4_single_join_kernel<128>, (size_t)kWarps * stages<4>() * stage_bytes<4>());
}

LLM_TRACE_EXPORT(attention_kv4_single)
