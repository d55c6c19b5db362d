// kv8_kernels.hip -- the 8-bit attention cache: new tokens into its pages, and
// attention over them.
#include "decode_launch.h"
#include "gemv_device.h"

#include <algorithm>
#include <math.h>

namespace dmc {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// The f32 of 2^(byte - 127); 255 is NaN, 0 is 2^-127, a subnormal.
__device__ __forceinline__ float e8m0(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// The byte of the least 2^e with amax <= 448 * 2^e, 448 = 1.75 * 2^8 being the
// largest e4m3 value; amax as its bits, finite.
__device__ __forceinline__ uint32_t e4m3_scale_byte(uint32_t amax) {
    const int e = (int)((amax + 0x1fffffu) >> 23) - 8;
    return (uint32_t)max(e, 0);
}

template <bool BF>
struct KvRow8 {  // 8 values of a row, any alignment of their type
    uint32_t u[BF ? 4 : 8];
    __device__ __forceinline__ void load(const void *p, int64_t at) {
        if constexpr (BF) {
            struct __attribute__((packed, aligned(2))) T { u32x4 v; };
            const u32x4 x = reinterpret_cast<const T *>(static_cast<const uint16_t *>(p) + at)->v;
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = x[i];
        } else {
            struct __attribute__((packed, aligned(4))) T { u32x4 v, w; };
            const T x = *reinterpret_cast<const T *>(static_cast<const float *>(p) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = x.v[i];
                u[4 + i] = x.w[i];
            }
        }
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (BF) return __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
        else return __uint_as_float(u[i]);
    }
    __device__ __forceinline__ uint32_t finite_max() const {  // infs and NaNs have no say in the scale
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t v = __float_as_uint(at(i)) & 0x7fffffffu;
            m = max(m, v < 0x7f800000u ? v : 0u);
        }
        return m;
    }
    // x 2^up in e4m3, to nearest even (the scaling is exact: one rounding); infs and NaNs become NaN
    __device__ __forceinline__ u32x2 codes(int up) const {
        u32x2 r = {0, 0};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            int c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(at(4 * w), up), ldexpf(at(4 * w + 1), up), 0, false);
            c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(at(4 * w + 2), up), ldexpf(at(4 * w + 3), up), c, true);
            r[w] = (uint32_t)c;
        }
        return r;
    }
};

__device__ __forceinline__ uint32_t rescale4(uint32_t u, int up) {  // 4 codes times 2^up; NaN stays NaN
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(a[0], up), ldexpf(a[1], up), 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(ldexpf(b[0], up), ldexpf(b[1], up), c, true);
    return (uint32_t)c;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

// Bytes of a dword that are among the tokens [lo, hi) at token t.
__device__ __forceinline__ uint32_t byte_mask(int t, int lo, int hi) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (t + i >= lo && t + i < hi) ? 0xffu << (8 * i) : 0u;
    return m;
}

// ---- append -------------------------------------------------------------------
//
// One workgroup per (page that gets tokens, head, sequence) and side, so that no
// two write the same page's codes or scale.  Positions [a, z) of the page are new;
// with a > 0 the page keeps the tokens before them, its scale only grows, and if
// it does their codes are rounded again (by a power of two: exact but where they
// become subnormal).  With a == 0 the scale is the new tokens' own.
//
// An item is 4 tokens x 8 dims, read once (a thread keeps its first item between
// the maximum and the codes; a page of more than NT items reads the others twice).
// A K item leaves as 8 bytes per token.  V lies transposed: an item's 4 x 4 bytes
// turn in registers into a dword per dim; a whole page passes through LDS, so that
// it leaves as one run of 16-byte stores, a part of one by dwords and bytes.
template <bool BF, int NT>
__global__ __launch_bounds__(NT) void kv_append_kernel(const KvAppend p) {
    extern __shared__ uint32_t turn[];
    __shared__ uint32_t part[NT / 64];
    const int b = blockIdx.z >> 1, head = blockIdx.y;
    const bool is_v = blockIdx.z & 1;
    const int D = p.c.dim, P = p.c.page, lgp = 31 - __clz(P), DC = D / 8;
    const int64_t start = p.b.starts[b];
    const int64_t len = p.b.lens[b];
    const int64_t count = min((int64_t)p.b.starts[b + 1] - start, (int64_t)p.b.max_new);
    const int64_t first = len - count;
    if (count <= 0 || first < 0) return;
    const int64_t slot = (first >> lgp) + blockIdx.x;
    if (slot * P >= len || slot >= p.b.width) return;
    const int64_t page = p.b.table[b * p.b.width + slot];
    if (page < 0 || page >= p.c.pages) return;
    const int a = (int)max((int64_t)0, first - slot * P), z = (int)min((int64_t)P, len - slot * P);
    const int64_t ld = is_v ? p.v_ld : p.k_ld;
    const void *src = is_v ? p.v : p.k;
    const int64_t row0 = (start + slot * P - first) * ld + (int64_t)head * D;  // of the page's token 0
    const int g0 = a >> 2, items = (((z + 3) >> 2) - g0) * DC;

    KvRow8<BF> it[4];
    auto load = [&](int i) {
        const int t = (g0 + i / DC) * 4, c = i % DC;
#pragma unroll
        for (int j = 0; j < 4; ++j) it[j].load(src, row0 + min(max(t + j, a), z - 1) * ld + c * 8);  // an edge's own row
    };
    uint32_t mag = 0;
    for (int i = threadIdx.x + (items - 1) / NT * NT; i >= 0; i -= NT) {  // the first item last: it stays
        if (i >= items) continue;
        load(i);
#pragma unroll
        for (int j = 0; j < 4; ++j) mag = max(mag, it[j].finite_max());
    }
    mag = wave_max(mag);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mag;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) mag = max(mag, part[w]);
    }
    uint8_t *scale = (is_v ? p.c.vs : p.c.ks) + page * p.c.heads + head;
    const uint32_t need = e4m3_scale_byte(mag), had = a > 0 ? *scale : 0u;
    const uint32_t byte = max(need, had);
    uint8_t *codes = (is_v ? p.c.v : p.c.k) + (page * p.c.heads + head) * (int64_t)(P * D);
    if (a > 0 && byte > had) {
        // V's dwords hold tokens 4 i .. 4 i + 3 of a dim; K's tokens before a come first
        uint32_t *w = reinterpret_cast<uint32_t *>(codes);
        const int n = is_v ? P * D / 4 : a * D / 4;
#pragma unroll 4
        for (int i = threadIdx.x * 4; i < n; i += NT * 4) {
            u32x4 u = *reinterpret_cast<const u32x4 *>(w + i);
            const int t = (i * 4) & (P - 1);
            if (is_v && t >= a) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t keep = is_v ? byte_mask(t + 4 * e, 0, a) : ~0u;
                u[e] = (rescale4(u[e], (int)had - (int)byte) & keep) | (u[e] & ~keep);
            }
            *reinterpret_cast<u32x4 *>(w + i) = u;
        }
        __syncthreads();  // before the new tokens' bytes beside them
    }
    if (NT > 64) __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *scale = (uint8_t)byte;
    const bool whole = is_v && a == 0 && z == P && p.turn;
    for (int i = threadIdx.x; i < items; i += NT) {
        if (i >= NT) load(i);
        const int t = (g0 + i / DC) * 4, c = i % DC;
        u32x2 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = it[j].codes(127 - (int)byte);
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (t + j >= a && t + j < z) *reinterpret_cast<u32x2 *>(codes + (t + j) * D + c * 8) = q[j];
            continue;
        }
        uint32_t d[8];  // dim e's tokens t .. t + 3
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t lo01 = __builtin_amdgcn_perm(q[1][w], q[0][w], 0x05010400u), lo23 = __builtin_amdgcn_perm(q[3][w], q[2][w], 0x05010400u);
            const uint32_t hi01 = __builtin_amdgcn_perm(q[1][w], q[0][w], 0x07030602u), hi23 = __builtin_amdgcn_perm(q[3][w], q[2][w], 0x07030602u);
            d[4 * w] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
            d[4 * w + 1] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
            d[4 * w + 2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
            d[4 * w + 3] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
        }
        if (whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e) turn[(c * 8 + e) * (P / 4 + 1) + (t >> 2)] = d[e];
        } else if (t >= a && t + 4 <= z) {
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<uint32_t *>(codes + (c * 8 + e) * P + t) = d[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (t + j >= a && t + j < z) codes[(c * 8 + e) * P + t + j] = (uint8_t)(d[e] >> (8 * j));
        }
    }
    if (whole) {
        __syncthreads();
        for (int i = threadIdx.x; i < P * D / 16; i += NT) {
            const int dim = i * 16 >> lgp, w = (i * 4) & (P / 4 - 1);
            const uint32_t *s = turn + dim * (P / 4 + 1) + w;
            *reinterpret_cast<u32x4 *>(codes + i * 16) = u32x4{s[0], s[1], s[2], s[3]};
        }
    }
}

// ---- attention ------------------------------------------------------------------
//
// For a query row q at position t of its sequence and the cached tokens j it sees
// (max(0, t - window + 1) <= j <= t, their page in the pool):
//   s_j = scale (q . K_j) 2^(ks - 127),  o = sum_j e^(s_j - m) V_j 2^(vs - 127) / sum_j e^(s_j - m)
// with the running maximum m and the sum in f32, in one pass over the tokens.
//
// The matrix cores take 16 tokens x 16 columns at a time, S' = K Q' and O' = V' P':
// codes are exact in bf16, and q and P enter as bf16 terms, one each where the
// caller's type is bf16, else three (cut, so that they add up to all 24 bits).  A
// column is a query row's term: 16 rows of bf16, or 4 rows x 4 terms (the last one
// zero) of f32, whose partial scores meet by two rotations within 16 lanes, and
// whose P terms are each formed in the column that multiplies them.
//
// In 64 tokens, lane 16 q + c of an S' tile holds column c of tokens 16 q + 4 j + i
// (tile j, register i): row r of tile j is token 16 (r / 4) + 4 j + r % 4.  So a
// lane's 16 tokens lie together, in one page with one scale (pages hold a multiple
// of 16), and are the k positions that the V' operand wants from one 16-byte read
// of a dim's tokens.
constexpr int kStep = 64;  // tokens per wave and step
constexpr int kMaxSplits = 256;  // workgroups along one sequence
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi) {  // 8 codes to bf16
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    return r;
}

__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Term t of f (0, 1, 2: 8 bits each, cut; 3: zero); an inf or a NaN is its first term alone.
__device__ __forceinline__ float term_of(float f, int t) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7f800000u) == 0x7f800000u) return t ? 0.0f : __uint_as_float((u & 0x7fffffu) ? u | 0x400000u : u);
    const float a = __uint_as_float(u & 0xffff0000u), r = f - a;
    const float b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
    return t == 0 ? a : t == 1 ? b : t == 2 ? r - b : 0.0f;
}

__device__ __forceinline__ uint32_t pair_cut(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

__device__ __forceinline__ uint32_t pair_near(float a, float b) {  // to nearest even
    const bf16x2_t r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ float ror_add(float v) {  // over columns c, c + 4, c + 8, c + 12 of 16
    v += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x128, 0xf, 0xf, false));
    v += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x124, 0xf, 0xf, false));
    return v;
}

// Bytes 0x01 where a code is NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {
    return (((v & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
}

// Which of a lane's values of a column (dim 16 d + 4 quad + i is bit 4 d + i) meet a NaN code among the
// tokens [lo, hi) that the column's row sees.  For the steps that some rows see in part: there a weight of
// zero must not meet a NaN, so NaN codes are taken out of the products, and only if there were any is this
// asked, once, at the end.
__device__ __forceinline__ uint64_t nan_dims(const KvAttend &p, const int32_t *table, int head, int quad, int lo, int hi) {
    uint64_t bits = 0;
    const int P = p.c.page, D = p.c.dim, lgp = 31 - __clz(P);
#pragma unroll 1
    for (int n = 0; n < D / 4; ++n) {
        const int dim = (n >> 2) * 16 + quad * 4 + (n & 3);
#pragma unroll 1
        for (int t = lo; t < hi; ++t) {
            const int64_t id = table[t >> lgp];
            if (id < 0 || id >= p.c.pages) continue;
            if ((p.c.v[((id * p.c.heads + head) * D + dim) * P + (t & (P - 1))] & 0x7f) == 0x7f) bits |= 1ull << n;
        }
    }
    return bits;
}

__device__ __forceinline__ float quads_max(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

struct KvPart {
    float *o;  // [splits][rows][dim]
    float *ml; // [splits][rows][2]
};

// Workgroups (column tile, token split), heads, sequences; 4 waves take steps of 64 tokens in turn.  A step's V is
// on its way to registers while its scores are formed, the next step's K from then on (into the registers
// that held this one's), so that each wave has 8 to 16 KB in flight without a second set of registers.
template <int D, bool BF>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv_rows_kernel(const KvAttend p, const KvPart part, int splits, int chunk,
                                                      int row_tiles, int64_t rows_total) {
    constexpr int R = BF ? 16 : 4;      // query rows per column tile
    constexpr int KS = D / 32;          // MFMA steps over dims
    constexpr int DT = D / 16;          // tiles of dims
    constexpr bool WIDE = KS % 2 == 0;  // K rows in 16-byte pieces (piece i of quad q: dims 64 i + 16 q on), else in 8
    constexpr int KP = WIDE ? KS / 2 : KS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int split = blockIdx.x / row_tiles, tile = blockIdx.x - split * row_tiles;
    const int head = blockIdx.y, b = blockIdx.z;
    const int group = p.q_heads / p.c.heads, P = p.c.page, lgp = 31 - __clz(P);
    const int64_t start = p.b.starts[b];
    const int count = (int)min((int64_t)p.b.starts[b + 1] - start, (int64_t)p.b.max_new);
    const int row0 = tile * R, rows = count * group;  // query rows of this head: token row / group, head row % group
    if (row0 >= rows) return;
    const int len = p.b.lens[b];
    const int here = min(R, rows - row0);
    // tokens that some row of the tile sees
    const int t_lo = len - count + row0 / group, t_hi = len - count + (row0 + here - 1) / group;
    const int most = (int)min((int64_t)INT32_MAX, p.b.width * P);
    const int see_hi = min(t_hi + 1, most);
    const int see_lo = p.window > 0 ? max(0, t_lo - p.window + 1) : 0;
    const int base = see_lo & ~(kStep - 1);
    const int from = base + split * chunk, to = split == splits - 1 ? see_hi : min(from + chunk, see_hi);
    if (split > 0 && from >= see_hi) return;  // the joining pass knows
    const int my = min(BF ? col : (col & 3), here - 1);          // this column's query row (the last one's for spare columns)
    const int64_t tok = start + (row0 + my) / group;
    const int qh = head * group + (row0 + my) % group;
    const int pos = len - count + (row0 + my) / group;
    const int vis_lo = p.window > 0 ? max(0, pos - p.window + 1) : 0, vis_hi = min(pos + 1, most);
    const int term = BF ? 0 : col >> 2;

    const int32_t *table = p.b.table + (int64_t)b * p.b.width;
    const float scale = p.scale * kLog2e;
    const int64_t page_bytes = (int64_t)P * D;
    auto page_of = [&](int t) -> int {  // no branch: past the table, its last entry is read and not taken
        const int id = table[min(t, most - 1) >> lgp];
        return t < most ? id : -1;
    };
    auto safe = [&](int id) -> int64_t { return id >= 0 && id < p.c.pages ? id : 0; };
    u32x4 kw[WIDE ? 4 * KP : 1];
    u32x2 k8[WIDE ? 1 : 4 * KP];
    // pk: the page of the 16 tokens that this lane's K rows (r / 4) lie in, pv: of this lane's own tokens
    auto load_k = [&](int t0, int pk) {
        const uint8_t *kp = p.c.k + (safe(pk) * p.c.heads + head) * page_bytes + (((t0 + 16 * (col >> 2)) & (P - 1)) + (col & 3)) * D;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                if constexpr (WIDE) kw[j * KP + i] = *reinterpret_cast<const u32x4 *>(kp + j * 4 * D + i * 64 + quad * 16);
                else k8[j * KP + i] = *reinterpret_cast<const u32x2 *>(kp + j * 4 * D + i * 32 + quad * 8);
            }
    };
    const int first = from + wave * kStep, tko = 16 * (col >> 2), tvo = 16 * quad;
    int pv = page_of(first + tvo), pk = page_of(first + 4 * kStep + tko), pv_next = page_of(first + 4 * kStep + tvo);
    load_k(first, page_of(first + tko));
    uint32_t ksb = p.c.ks[safe(pv) * p.c.heads + head], vsb = p.c.vs[safe(pv) * p.c.heads + head];

    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int dim = WIDE ? (s >> 1) * 64 + quad * 16 + (s & 1) * 8 : s * 32 + quad * 8;
        const int64_t at = tok * p.q_ld + (int64_t)qh * D + dim;
        if constexpr (BF) {
            struct __attribute__((packed, aligned(2))) T8 { u32x4 v; };
            qf[s] = reinterpret_cast<const T8 *>(static_cast<const uint16_t *>(p.q) + at)->v;
        } else {
            const float *f = static_cast<const float *>(p.q) + at;
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[s][i] = pair_cut(term_of(f[2 * i], term), term_of(f[2 * i + 1], term));
        }
    }

    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, sum = 0.0f;
    uint32_t nans = 0;

    for (int t0 = first; t0 < to; t0 += 4 * kStep) {
        const int tv = t0 + tvo;
        const bool in = pv >= 0 && pv < p.c.pages;
        u32x4 vw[DT];
        const uint8_t *vp = p.c.v + (safe(pv) * p.c.heads + head) * page_bytes + col * P + (tv & (P - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d) vw[d] = *reinterpret_cast<const u32x4 *>(vp + d * 16 * P);
        const float ks = e8m0(ksb) * scale, vs = e8m0(vsb);
        float s[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                if constexpr (WIDE) {
                    const u32x4 w = kw[j * KP + i];
                    c = mma(widen8(w[0], w[1]), qf[2 * i], c);
                    c = mma(widen8(w[2], w[3]), qf[2 * i + 1], c);
                } else {
                    const u32x2 w = k8[j * KP + i];
                    c = mma(widen8(w[0], w[1]), qf[i], c);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * j + i] = c[i];
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(t0 + 4 * kStep, pk);  // past the end: some page's codes, not used
        pv = pv_next;
        ksb = p.c.ks[safe(pv) * p.c.heads + head];
        vsb = p.c.vs[safe(pv) * p.c.heads + head];
        pk = page_of(t0 + 8 * kStep + tko);
        pv_next = page_of(t0 + 8 * kStep + tvo);
        const bool whole = t0 >= see_lo && t0 >= t_hi - (p.window > 0 ? p.window - 1 : INT32_MAX - 1) &&
                           t0 + kStep - 1 <= t_lo && t0 + kStep <= most;
        const bool every = __builtin_amdgcn_ballot_w64(!in) == 0 && whole;  // nothing masked in this step
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (!BF) s[i] = ror_add(s[i]);
            s[i] *= ks;
        }
        if (!every) {
            // codes that no row sees read as zero, and so do NaN codes, for now (nan_dims)
            const int lo = in ? vis_lo - tv : 16, hi = vis_hi - tv;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
            uint32_t keep[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) keep[i] = byte_mask(tv + 4 * i, see_lo, in ? see_hi : 0);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t u = vw[d][i] & keep[i], bad = nan_bytes(u);
                    vw[d][i] = u & ~(bad * 0xffu);
                    nans |= bad;
                }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        top = quads_max(top);
        // the maximum moves only when it has grown by 2^8: weights stay within f32 and bf16 meanwhile
        const bool grow = top > m + 8.0f || (m == -INFINITY && top > -INFINITY);
        if (__builtin_amdgcn_ballot_w64(grow)) {
            const float m2 = grow ? top : m;
            const float alpha = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m2);
            m = m2;
            sum *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float add = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
            add += s[i];
            s[i] *= vs;
        }
        sum += add;
        u32x4 pf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = s[8 * u + 2 * i], c = s[8 * u + 2 * i + 1];
                pf[u][i] = BF ? pair_near(a, c) : pair_cut(term_of(a, term), term_of(c, term));
            }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const u32x4 v = vw[d];
            o[d] = mma(widen8(v[0], v[1]), pf[0], o[d]);
            o[d] = mma(widen8(v[2], v[3]), pf[1], o[d]);
        }
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if constexpr (!BF) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] = ror_add(o[d][i]);
    }
    if (__builtin_amdgcn_ballot_w64(nans != 0)) {
        const uint64_t bits = nan_dims(p, table, head, quad, max(from, vis_lo), min(to, vis_hi));
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] = (bits >> (4 * d + i)) & 1 ? NAN : o[d][i];
    }

    // join the 4 waves: lanes of the tile's rows put their part down, wave w takes dims w * D / 4 ..
    __shared__ float ml[4][16][2];
    __shared__ float ow[4][R][D + 4];
    if (quad == 0) {
        ml[wave][col][0] = m;
        ml[wave][col][1] = sum;
    }
    if (col < R) {
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(&ow[wave][col][d * 16 + quad * 4]) = o[d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < here * D; i += 256) {
        const int row = i / D, d = i - row * D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][row][0]);
        // a NaN score leaves its row's sum NaN, whatever the maximum
        const float ref = top == -INFINITY ? 0.0f : top;
        float val = 0.0f, tot = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w][row][0] - ref);
            val += f * ow[w][row][d];
            tot += f * ml[w][row][1];
        }
        const int64_t t = start + (row0 + row) / group;
        const int h = head * group + (row0 + row) % group;
        if (splits == 1) {
            const float r = tot == 0.0f ? 0.0f : val / tot;  // nothing seen: zero
            const int64_t at = t * p.out_ld + (int64_t)h * D + d;
            if constexpr (BF) static_cast<__bf16 *>(p.out)[at] = (__bf16)r;
            else static_cast<float *>(p.out)[at] = r;
        } else {
            const int64_t at = ((int64_t)split * rows_total + (int64_t)b * p.b.max_new + (row0 + row) / group) * p.q_heads + h;
            part.o[at * D + d] = val;
            if (d == 0) {
                part.ml[at * 2] = top;
                part.ml[at * 2 + 1] = tot;
            }
        }
    }
}

// ---- attention, tiles of query rows ----------------------------------------------
//
// Prompts: a workgroup of 4 waves owns 64 * CT query rows of one cache head (tokens x
// the head's group of query heads) and walks the tokens 64 at a time.  The codes go to
// LDS as they are, without passing through registers, one step ahead; every wave widens
// them for its own CT column tiles.  f32 rows take one MFMA per term of q (3) and of
// the weights (3) instead of a column per term, so that a weight is computed once.
//
// 16-byte pieces of a K row (a dim's tokens of V) are stored in an order that depends on
// the row, so that the 8 lanes that read at a time meet different banks.
template <int D>
struct KvTile {
    static constexpr int KC = D / 16;                     // pieces of a K row
    static constexpr int K_BYTES = kStep * D, BYTES = 2 * kStep * D;
    static constexpr int PASSES = (kStep * KC + 255) / 256;  // pieces per thread and side
    static __device__ __forceinline__ int k_slot(int t, int c) {
        return KC == 6 ? c : c ^ (((t & 3) | ((t >> 2) & 4)) & (KC >= 8 ? 7 : 3));
    }
    static __device__ __forceinline__ int v_slot(int d, int c) { return c ^ ((d >> 1) & 3); }
};

__device__ __forceinline__ void lds_copy16(const void *g, char *l) {  // lane i's 16 bytes to l + 16 i
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)g,
                                     (__attribute__((address_space(3))) uint32_t *)l, 16, 0, 0);
}

template <int D, bool BF, int CT>
__global__ __launch_bounds__(256, D == 256 && !BF ? 1 : 2) void kv_tiles_kernel(const KvAttend p, const KvPart part, int splits, int chunk,
                                                          int row_tiles, int64_t rows_total) {
    using T = KvTile<D>;
    constexpr int PL = BF ? 1 : 3;  // terms of q and of the weights
    constexpr int KS = D / 32, DT = D / 16, LB = D / 4, R = 64 * CT;
    __shared__ __attribute__((aligned(16))) char lds[2][T::BYTES];
    __shared__ int nans;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    // heads turn fastest: with 8 of them each XCD keeps one head's codes in its L2
    const int head = blockIdx.x % p.c.heads, rest = blockIdx.x / p.c.heads, b = blockIdx.y;
    const int split = rest / row_tiles, tile = row_tiles - 1 - (rest - split * row_tiles);  // the longest first
    const int group = p.q_heads / p.c.heads, P = p.c.page, lgp = 31 - __clz(P);
    const int64_t start = p.b.starts[b];
    const int count = (int)min((int64_t)p.b.starts[b + 1] - start, (int64_t)p.b.max_new);
    const int row0 = tile * R, rows = count * group;
    if (row0 >= rows) return;
    const int len = p.b.lens[b];
    const int here = min(R, rows - row0);
    const int t_lo = len - count + row0 / group, t_hi = len - count + (row0 + here - 1) / group;
    const int most = (int)min((int64_t)INT32_MAX, p.b.width * P);
    const int see_hi = min(t_hi + 1, most);
    const int see_lo = p.window > 0 ? max(0, t_lo - p.window + 1) : 0;
    const int from = (see_lo & ~(kStep - 1)) + split * chunk;
    const int to = split == splits - 1 ? see_hi : min(from + chunk, see_hi);
    if (split > 0 && from >= see_hi) return;

    u32x4 qf[CT][PL][KS];
    int vis_lo[CT], vis_hi[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int my = min(row0 + (wave * CT + c) * 16 + col, rows - 1);
        const int pos = len - count + my / group;
        vis_lo[c] = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        vis_hi[c] = min(pos + 1, most);
        const int64_t q0 = (start + my / group) * p.q_ld + (int64_t)(head * group + my % group) * D + quad * LB;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (BF) {
                struct __attribute__((packed, aligned(2))) T8 { u32x4 v; };
                qf[c][0][s] = reinterpret_cast<const T8 *>(static_cast<const uint16_t *>(p.q) + q0 + s * 8)->v;
            } else {
                const float *f = static_cast<const float *>(p.q) + q0 + s * 8;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < PL; ++t) qf[c][t][s][i] = pair_cut(term_of(f[2 * i], t), term_of(f[2 * i + 1], t));
            }
        }
    }

    const int32_t *table = p.b.table + (int64_t)b * p.b.width;
    const float scale = p.scale * kLog2e;
    const int64_t page_bytes = (int64_t)P * D;
    auto page_of = [&](int t) -> int {  // no branch: past the table, its last entry is read and not taken
        const int id = table[min(t, most - 1) >> lgp];
        return t < most ? id : -1;
    };
    auto safe = [&](int id) -> int64_t { return id >= 0 && id < p.c.pages ? id : 0; };

    // This thread's pieces of a step: K token rows kt[], V's 16 tokens vc.
    int kt[T::PASSES], kc[T::PASSES], vd[T::PASSES];
    const int vslot = threadIdx.x & 3, vc = vslot ^ ((threadIdx.x >> 3) & 3);
#pragma unroll
    for (int i = 0; i < T::PASSES; ++i) {
        const int at = i * 256 + threadIdx.x;
        kt[i] = at / T::KC;
        kc[i] = T::k_slot(kt[i], at % T::KC);
        vd[i] = at >> 2;
    }
    int kid[T::PASSES], vid;
    auto ids = [&](int t0) {
#pragma unroll
        for (int i = 0; i < T::PASSES; ++i) kid[i] = kt[i] < kStep ? page_of(t0 + kt[i]) : -1;
        vid = page_of(t0 + 16 * vc);
    };
    auto fetch = [&](int t0, char *buf) {
#pragma unroll
        for (int i = 0; i < T::PASSES; ++i) {
            if (kStep * T::KC % 256 && i == T::PASSES - 1 && wave * 64 >= kStep * T::KC % 256) break;
            const uint8_t *k = p.c.k + (safe(kid[i]) * p.c.heads + head) * page_bytes + ((t0 + kt[i]) & (P - 1)) * D + kc[i] * 16;
            lds_copy16(k, buf + (i * 256 + wave * 64) * 16);
        }
        const uint8_t *v = p.c.v + (safe(vid) * p.c.heads + head) * page_bytes + ((t0 + 16 * vc) & (P - 1));
#pragma unroll
        for (int i = 0; i < T::PASSES; ++i) {
            if (kStep * T::KC % 256 && i == T::PASSES - 1 && wave * 64 >= kStep * T::KC % 256) break;
            lds_copy16(v + vd[i] * P, buf + T::K_BYTES + (i * 256 + wave * 64) * 16);
        }
    };

    f32x4 o[CT][DT];
    float m[CT], sum[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        m[c] = -INFINITY;
        sum[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[c][d] = f32x4{0, 0, 0, 0};
    }
    // where this lane's K row pieces (tokens 4 j on, piece i by its low bits) and V pieces lie
    const int k_tok = 16 * (col >> 2) + (col & 3);
    const int k_at = k_tok * D, k_piece = KS % 2 == 0 ? T::k_slot(k_tok, quad * (KS / 2)) * 16 : 0;
    const int v_at = (col * 4 + T::v_slot(col, quad)) * 16;
    int buf = 0;
    if (threadIdx.x == 0) nans = 0;
    if (from < to) {
        ids(from);
        fetch(from, lds[0]);
        ids(from + kStep);
    }
    // this lane's 16 tokens: their page and its scales, a step ahead of their use
    int own = page_of(from + 16 * quad), own_next = page_of(from + kStep + 16 * quad);
    uint32_t ksb = p.c.ks[safe(own) * p.c.heads + head], vsb = p.c.vs[safe(own) * p.c.heads + head];
    for (int t0 = from; t0 < to; t0 += kStep) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t0 + kStep < to) fetch(t0 + kStep, lds[buf ^ 1]);
        ids(t0 + 2 * kStep);
        const bool in = own >= 0 && own < p.c.pages;
        const float ks = e8m0(ksb) * scale;
        const uint32_t vb = vsb;
        own = own_next;
        own_next = page_of(t0 + 2 * kStep + 16 * quad);
        ksb = p.c.ks[safe(own) * p.c.heads + head];
        vsb = p.c.vs[safe(own) * p.c.heads + head];
        const int tv = t0 + 16 * quad;
        const bool whole = t0 >= see_lo && t0 >= t_hi - (p.window > 0 ? p.window - 1 : INT32_MAX - 1) &&
                           t0 + kStep - 1 <= t_lo && t0 + kStep <= most;
        const bool every = __builtin_amdgcn_ballot_w64(!in) == 0 && whole;  // nothing masked in this step
        if (!every) {
            // V codes that no row sees read as zero, and so do NaN codes, for now (nan_dims); every wave
            // sees the same four pages, so the whole workgroup is here
            const int t = t0 + 16 * vc;
            const int id = page_of(t);
            const int hi = id >= 0 && id < p.c.pages ? see_hi : 0;
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < T::PASSES; ++i) {
                if (i * 256 + (int)threadIdx.x >= kStep * T::KC) break;
                uint32_t *v = reinterpret_cast<uint32_t *>(lds[buf] + T::K_BYTES + (i * 256 + threadIdx.x) * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t u = v[e] & byte_mask(t + 4 * e, see_lo, hi), n = nan_bytes(u);
                    bad |= n;
                    v[e] = u & ~(n * 0xffu);
                }
            }
            if (bad) nans = 1;
            __syncthreads();
        }
        const char *kb = lds[buf] + k_at, *vl = lds[buf] + T::K_BYTES + v_at;

        float s[CT][16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j) __builtin_amdgcn_sched_barrier(0);
            u32x2 w[KS];
            if constexpr (KS % 2 == 0) {
#pragma unroll
                for (int i = 0; i < KS / 2; ++i) {
                    const u32x4 x = *reinterpret_cast<const u32x4 *>(kb + j * 4 * D + (k_piece ^ (i * 16)));
                    w[2 * i] = u32x2{x[0], x[1]};
                    w[2 * i + 1] = u32x2{x[2], x[3]};
                }
            } else {
#pragma unroll
                for (int i = 0; i < KS; ++i) w[i] = *reinterpret_cast<const u32x2 *>(kb + j * 4 * D + quad * LB + i * 8);
            }
            f32x4 acc[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[c] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const u32x4 a = widen8(w[i][0], w[i][1]);
#pragma unroll
                for (int t2 = PL - 1; t2 >= 0; --t2)
#pragma unroll
                    for (int c = 0; c < CT; ++c) acc[c] = mma(a, qf[c][t2][i], acc[c]);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[c][4 * j + i] = acc[c][i];
        }

        __builtin_amdgcn_sched_barrier(0);
        // V's scale enters the weight through the exponent, but where that could leave the exponent's range
        const bool fold = vb >= 67 && vb <= 187;
        const float shift = fold ? (float)((int)vb - 127) : 0.0f;
        const float unfold = fold ? e8m0(254 - vb) : 1.0f;
        const bool plain = __builtin_amdgcn_ballot_w64(!fold) != 0;
        u32x4 pf[CT][PL][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            if (!every) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[c][i] = (in && tv + i >= vis_lo[c] && tv + i < vis_hi[c]) ? s[c][i] : -INFINITY;
            }
            float top = s[c][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, s[c][i]);
            top = quads_max(top * ks);
            // the maximum moves only when it has grown by 2^8: weights stay within f32 and bf16 meanwhile
            const bool grow = top > m[c] + 8.0f || (m[c] == -INFINITY && top > -INFINITY);
            if (__builtin_amdgcn_ballot_w64(grow)) {
                const float m2 = grow ? top : m[c];
                const float alpha = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[c] - m2);
                m[c] = m2;
                sum[c] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[c][d] *= alpha;
            }
            const float off = shift - (m[c] == -INFINITY ? 0.0f : m[c]);
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[c][i] = __builtin_amdgcn_exp2f(fmaf(s[c][i], ks, off));
                add += s[c][i];
            }
            sum[c] = fmaf(add, unfold, sum[c]);
            if (plain) {
                const float vs = fold ? 1.0f : e8m0(vb);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[c][i] *= vs;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = s[c][8 * u + 2 * i], y = s[c][8 * u + 2 * i + 1];
                    if constexpr (BF) {
                        pf[c][0][u][i] = pair_near(x, y);
                    } else {
#pragma unroll
                        for (int t = 0; t < PL; ++t) pf[c][t][u][i] = pair_cut(term_of(x, t), term_of(y, t));
                    }
                }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(vl + d * 1024);
            const u32x4 a0 = widen8(v[0], v[1]), a1 = widen8(v[2], v[3]);
#pragma unroll
            for (int t = PL - 1; t >= 0; --t)
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    o[c][d] = mma(a0, pf[c][t][0], o[c][d]);
                    o[c][d] = mma(a1, pf[c][t][1], o[c][d]);
                }
        }
        buf ^= 1;
    }

    __syncthreads();
    if (nans) {
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const uint64_t bits = nan_dims(p, table, head, quad, max(from, vis_lo[c]), min(to, vis_hi[c]));
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][d][i] = (bits >> (4 * d + i)) & 1 ? NAN : o[c][d][i];
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        sum[c] += __shfl_xor(sum[c], 16);
        sum[c] += __shfl_xor(sum[c], 32);
        const int r = row0 + (wave * CT + c) * 16 + col;
        if (r >= rows) continue;
        const int h = head * group + r % group;
        if (splits == 1) {
            const float inv = sum[c] == 0.0f ? 0.0f : 1.0f / sum[c];  // nothing seen: zero
            const int64_t at = (start + r / group) * p.out_ld + (int64_t)h * D + quad * 4;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (BF) static_cast<__bf16 *>(p.out)[at + d * 16 + i] = (__bf16)(o[c][d][i] * inv);
                    else static_cast<float *>(p.out)[at + d * 16 + i] = o[c][d][i] * inv;
                }
        } else {
            const int64_t at = ((int64_t)split * rows_total + (int64_t)b * p.b.max_new + r / group) * p.q_heads + h;
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(part.o + at * D + d * 16 + quad * 4) = o[c][d];
            if (quad == 0) {
                part.ml[at * 2] = m[c];
                part.ml[at * 2 + 1] = sum[c];
            }
        }
    }
}

// Joins the token splits of one query row and head: wave w takes every fourth split, a lane dims lane, lane + 64, ..
template <bool BF>
__global__ __launch_bounds__(256) void kv_join_kernel(const KvAttend p, const KvPart part, int splits, int chunk,
                                                      int rows_per_tile, int64_t rows_total) {
    const int b = blockIdx.z, h = blockIdx.y, D = p.c.dim;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int group = p.q_heads / p.c.heads;
    const int64_t start = p.b.starts[b];
    const int count = (int)min((int64_t)p.b.starts[b + 1] - start, (int64_t)p.b.max_new);
    const int i = blockIdx.x;
    if (i >= count) return;
    // the splits that this row's tile wrote
    const int r = i * group + h % group, row0 = r - r % rows_per_tile, here = min(rows_per_tile, count * group - row0);
    const int len = p.b.lens[b];
    const int t_lo = len - count + row0 / group, t_hi = len - count + (row0 + here - 1) / group;
    const int see_hi = min(t_hi + 1, (int)min((int64_t)INT32_MAX, p.b.width * p.c.page));
    const int see_lo = p.window > 0 ? max(0, t_lo - p.window + 1) : 0;
    const int span = see_hi - (see_lo & ~(kStep - 1));
    const int used = max(1, min(splits, (span + chunk - 1) / chunk));
    const int64_t at = ((int64_t)b * p.b.max_new + i) * p.q_heads + h, step = rows_total * p.q_heads;
    // the splits' weights once, then their sums with independent loads
    __shared__ float f[kMaxSplits];
    float top = -INFINITY;
    for (int s = lane; s < used; s += 64) top = fmaxf(top, part.ml[(at + s * step) * 2]);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -INFINITY ? 0.0f : top;
    float tot = 0.0f;
    for (int s = threadIdx.x; s < used; s += 256) {
        f[s] = __builtin_amdgcn_exp2f(part.ml[(at + s * step) * 2] - ref);
        tot += f[s] * part.ml[(at + s * step) * 2 + 1];
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) tot += __shfl_xor(tot, d);
    __syncthreads();
    float val[4] = {0, 0, 0, 0};
    const float *po = part.o + at * D + lane;
    for (int s = wave; s < used; s += 32) {
        float v[8][4];
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[u][j] = s + 4 * u < used && lane + 64 * j < D ? po[(s + 4 * u) * step * D + 64 * j] : 0.0f;
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) val[j] += (s + 4 * u < used ? f[s + 4 * u] : 0.0f) * v[u][j];
    }
    __shared__ float vals[4][256], tots[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vals[wave][lane + 64 * j] = val[j];
    if (lane == 0) tots[wave] = tot;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    tot = (tots[0] + tots[1]) + (tots[2] + tots[3]);
    const float sum = (vals[0][d] + vals[1][d]) + (vals[2][d] + vals[3][d]);
    const float o = tot == 0.0f ? 0.0f : sum / tot;
    const int64_t to = (start + i) * p.out_ld + (int64_t)h * D + d;
    if constexpr (BF) static_cast<__bf16 *>(p.out)[to] = (__bf16)o;
    else static_cast<float *>(p.out)[to] = o;
}

// Column tiles per wave: as many as 256 registers hold.
template <int D, bool BF>
constexpr int kTiles = BF && D <= 128 ? 2 : 1;

// Query rows of one head that a workgroup owns.
int tile_rows(const KvAttend &p, int kind) {
    if (kind == 0) return p.bf16 ? 16 : 4;
    return 64 * (p.bf16 && p.c.dim <= 128 ? 2 : 1);
}

template <bool BF>
hipError_t attend(const KvAttend &p, const KvPlan &pl, void *workspace, hipStream_t stream) {
    const int group = p.q_heads / p.c.heads, R = tile_rows(p, pl.kind);
    const int row_tiles = (p.b.max_new * group + R - 1) / R;
    const int64_t rows_total = (int64_t)p.b.batch * p.b.max_new;
    KvPart part{};
    part.o = static_cast<float *>(workspace);
    part.ml = part.o + (size_t)pl.splits * rows_total * p.q_heads * p.c.dim;
    const dim3 rows_grid((unsigned)(pl.splits * row_tiles), (unsigned)p.c.heads, (unsigned)p.b.batch);
    const dim3 tiles_grid((unsigned)(pl.splits * row_tiles * p.c.heads), (unsigned)p.b.batch);
#define DMC_DIM(N)                                                                                                        \
    case N:                                                                                                               \
        if (pl.kind == 0)                                                                                                 \
            kv_rows_kernel<N, BF><<<rows_grid, dim3(256), 0, stream>>>(p, part, pl.splits, pl.chunk, row_tiles, rows_total); \
        else                                                                                                              \
            kv_tiles_kernel<N, BF, kTiles<N, BF>>                                                                         \
                <<<tiles_grid, dim3(256), 0, stream>>>(p, part, pl.splits, pl.chunk, row_tiles, rows_total);              \
        break;
    switch (p.c.dim) {
        DMC_DIM(64)
        DMC_DIM(96)
        DMC_DIM(128)
        DMC_DIM(256)
    }
#undef DMC_DIM
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && pl.splits > 1) {
        kv_join_kernel<BF><<<dim3((unsigned)p.b.max_new, (unsigned)p.q_heads, (unsigned)p.b.batch), dim3(256), 0, stream>>>(
            p, part, pl.splits, pl.chunk, R, rows_total);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

bool kv_dim_served(int64_t dim) { return dim == 64 || dim == 96 || dim == 128 || dim == 256; }

hipError_t launch_kv_append(const KvAppend &args, hipStream_t stream) {
    KvAppend p = args;
    const int P = p.c.page, D = p.c.dim;
    const dim3 grid((unsigned)((p.b.max_new + 2 * P - 2) / P), (unsigned)p.c.heads, (unsigned)p.b.batch * 2);
    // few tokens are one wave's work (up to 8 of 4 x 8 values in 64 threads): no barrier between waves
    const bool few = p.b.max_new <= 4;
    const size_t lds = (size_t)D * (P / 4 + 1) * 4;
    p.turn = !few && lds <= 64 * 1024 - 64;
    const size_t use = p.turn ? lds : 0;
    if (few && p.bf16) kv_append_kernel<true, 64><<<grid, dim3(64), use, stream>>>(p);
    else if (few) kv_append_kernel<false, 64><<<grid, dim3(64), use, stream>>>(p);
    else if (p.bf16) kv_append_kernel<true, 256><<<grid, dim3(256), use, stream>>>(p);
    else kv_append_kernel<false, 256><<<grid, dim3(256), use, stream>>>(p);
    return hipGetLastError();
}

KvPlan plan_kv(const KvAttend &p, int num_cus) {
    KvPlan pl{};
    const int group = p.q_heads / p.c.heads;
    pl.kind = p.b.max_new * group > 16 ? 1 : 0;
    const int R = tile_rows(p, pl.kind);
    const int64_t tiles = (int64_t)((p.b.max_new * group + R - 1) / R) * p.c.heads * p.b.batch;
    const int64_t unit = pl.kind ? kStep : 4 * kStep;  // tokens of a workgroup's step
    int64_t span = p.b.max_len;
    if (p.window > 0) span = std::min<int64_t>(span, p.window + R + kStep);
    const int64_t units = std::max<int64_t>(1, (span + unit - 1) / unit);
    const int64_t want = std::max<int64_t>(1, (pl.kind ? 2 : 8) * num_cus / std::max<int64_t>(1, tiles));
    // steps per workgroup: a split of few costs more in its partial results than it saves
    const int64_t per = std::max<int64_t>((units + want - 1) / want, std::max<int64_t>(pl.kind ? 8 : 4, (units + kMaxSplits - 1) / kMaxSplits));
    pl.chunk = (int)(per * unit);
    pl.splits = (int)((units + per - 1) / per);
    if (pl.splits > 1)
        pl.workspace_bytes = (size_t)pl.splits * p.b.batch * p.b.max_new * p.q_heads * (p.c.dim + 2) * 4;
    return pl;
}

hipError_t launch_kv_attend(const KvAttend &p, const KvPlan &pl, void *workspace, hipStream_t stream) {
    return p.bf16 ? attend<true>(p, pl, workspace, stream) : attend<false>(p, pl, workspace, stream);
}

}  // namespace dmc
