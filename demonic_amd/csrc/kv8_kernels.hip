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

// Magnitude bits that count for a page's scale: infs and NaNs have no code but NaN and leave it alone.
__device__ __forceinline__ uint32_t finite_mag(float f) {
    const uint32_t u = __float_as_uint(f) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// x 2^(127 - byte) in e4m3, to nearest even (exact scaling, one rounding); infs and NaNs become NaN.
__device__ __forceinline__ uint32_t to_e4m3(float x, int byte) {
    const float f = ldexpf(x, 127 - byte);
    const uint32_t c = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 255u;
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 0x7fu : c;
}

__device__ __forceinline__ float from_e4m3(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

template <bool BF>
__device__ __forceinline__ float load1(const void *p, int64_t at) {
    if constexpr (BF) return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[at] << 16);
    else return static_cast<const float *>(p)[at];
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
    return v;
}

// ---- append -------------------------------------------------------------------
//
// One workgroup per (page that gets tokens, head, sequence) and side, so that no
// two write the same page's codes or scale.  Positions [a, z) of the page are new;
// with a > 0 the page keeps the tokens before them, its scale only grows, and if
// it does their codes are rounded again (by a power of two: exact but where they
// become subnormal).  With a == 0 the scale is the new tokens' own.
template <bool BF>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppend p) {
    const int b = blockIdx.z >> 1, head = blockIdx.y;
    const bool is_v = blockIdx.z & 1;
    const int D = p.c.dim, P = p.c.page;
    const int64_t start = p.b.starts[b];
    const int64_t len = p.b.lens[b];
    const int64_t count = min((int64_t)p.b.starts[b + 1] - start, (int64_t)p.b.max_new);
    const int64_t first = len - count;
    if (count <= 0 || first < 0) return;
    const int64_t slot = first / P + blockIdx.x;
    if (slot * P >= len || slot >= p.b.width) return;
    const int64_t page = p.b.table[b * p.b.width + slot];
    if (page < 0 || page >= p.c.pages) return;
    const int a = (int)max((int64_t)0, first - slot * P), z = (int)min((int64_t)P, len - slot * P);
    const int n = (z - a) * D;
    const int64_t ld = is_v ? p.v_ld : p.k_ld;
    const void *src = is_v ? p.v : p.k;
    const int64_t row0 = (start + slot * P + a - first) * ld + (int64_t)head * D;

    __shared__ uint32_t part[4];
    uint32_t mag = 0;
    for (int i = threadIdx.x; i < n; i += 256) mag = max(mag, finite_mag(load1<BF>(src, row0 + (int64_t)(i / D) * ld + i % D)));
    mag = wave_max(mag);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mag;
    __syncthreads();
    mag = max(max(part[0], part[1]), max(part[2], part[3]));
    uint8_t *scale = (is_v ? p.c.vs : p.c.ks) + page * p.c.heads + head;
    const uint32_t need = e4m3_scale_byte(mag), had = a > 0 ? *scale : 0u;
    const uint32_t byte = max(need, had);
    uint8_t *codes = (is_v ? p.c.v : p.c.k) + (page * p.c.heads + head) * (int64_t)(P * D);
    __syncthreads();
    if (threadIdx.x == 0) *scale = (uint8_t)byte;
    const int ts = is_v ? 1 : D, ds = is_v ? P : 1;  // strides of a token and a dim
    if (a > 0 && byte > had) {
        for (int i = threadIdx.x; i < a * D; i += 256) {
            uint8_t *c = codes + (i / D) * ts + (i % D) * ds;
            const uint32_t u = *c;
            const uint32_t r = to_e4m3(from_e4m3(u), (int)(127 + byte - had));
            *c = (uint8_t)((u & 0x7f) == 0x7f ? u : r);
        }
    }
    for (int i = threadIdx.x; i < n; i += 256)
        codes[(a + i / D) * ts + (i % D) * ds] = (uint8_t)to_e4m3(load1<BF>(src, row0 + (int64_t)(i / D) * ld + i % D), (int)byte);
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

// Bytes of a dword that are among the token range [lo, hi) at token t.
__device__ __forceinline__ uint32_t byte_mask(int t, int lo, int hi) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (t + i >= lo && t + i < hi) ? 0xffu << (8 * i) : 0u;
    return m;
}

// Bytes 0x01 where a code is NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {
    return (((v & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
}

struct KvPart {
    float *o;  // [splits][rows][dim]
    float *ml; // [splits][rows][2]
};

// Workgroups (column tile, token split), heads, sequences; 4 waves take steps of 64 tokens in turn.
template <int D, bool BF>
__global__ __launch_bounds__(256) void kv_rows_kernel(const KvAttend p, const KvPart part, int splits, int chunk,
                                                      int row_tiles, int64_t rows_total) {
    constexpr int R = BF ? 16 : 4;      // query rows per column tile
    constexpr int KS = D / 32;          // MFMA steps over dims
    constexpr int DT = D / 16;          // tiles of dims
    constexpr int LB = D / 4;           // dims of a lane of a K row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int split = blockIdx.x / row_tiles, tile = blockIdx.x - split * row_tiles;
    const int head = blockIdx.y, b = blockIdx.z;
    const int group = p.q_heads / p.c.heads, P = p.c.page;
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

    u32x4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int64_t at = tok * p.q_ld + (int64_t)qh * D + quad * LB + s * 8;
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
    const int32_t *table = p.b.table + (int64_t)b * p.b.width;
    const float scale = p.scale * kLog2e;
    const int64_t page_bytes = (int64_t)P * D;

    for (int t0 = from + wave * kStep; t0 < to; t0 += 4 * kStep) {
        // the page of 16 tokens, for a K row (r / 4 of 4) and for this lane's own tokens
        const int tk = t0 + 16 * (col >> 2), tv = t0 + 16 * quad;
        const int64_t pk_raw = tk < most ? table[tk / P] : -1, pv_raw = tv < most ? table[tv / P] : -1;
        const bool in_v = pv_raw >= 0 && pv_raw < p.c.pages;
        const int64_t pk = pk_raw >= 0 && pk_raw < p.c.pages ? pk_raw : 0, pv = in_v ? pv_raw : 0;
        const uint8_t *kp = p.c.k + (pk * p.c.heads + head) * page_bytes + (int64_t)(tk % P + (col & 3)) * D + quad * LB;
        const uint8_t *vp = p.c.v + (pv * p.c.heads + head) * page_bytes + (int64_t)col * P + tv % P;
        const float ks = e8m0(p.c.ks[pv * p.c.heads + head]) * scale, vs = e8m0(p.c.vs[pv * p.c.heads + head]);
        float s[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x2 kw[KS];
#pragma unroll
            for (int i = 0; i < KS; ++i) kw[i] = *reinterpret_cast<const u32x2 *>(kp + j * 4 * D + i * 8);
            f32x4 c = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KS; ++i) c = mma(widen8(kw[i][0], kw[i][1]), qf[i], c);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * j + i] = c[i];
        }
        const bool whole = t0 >= see_lo && t0 >= t_hi - (p.window > 0 ? p.window - 1 : INT32_MAX - 1) &&
                           t0 + kStep - 1 <= t_lo && t0 + kStep <= most;
        const bool every = __builtin_amdgcn_ballot_w64(!in_v) == 0 && whole;  // nothing masked in this step
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (!BF) s[i] = ror_add(s[i]);
            s[i] *= ks;
            if (!every) s[i] = (in_v && tv + i >= vis_lo && tv + i < vis_hi) ? s[i] : -INFINITY;
            top = fmaxf(top, s[i]);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m2 = fmaxf(m, top);
        const float ref = m2 == -INFINITY ? 0.0f : m2;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = m2;
        float add = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
            add += s[i];
            s[i] *= vs;
        }
        sum = sum * alpha + add;
        u32x4 pf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = s[8 * u + 2 * i], c = s[8 * u + 2 * i + 1];
                pf[u][i] = BF ? pair_near(a, c) : pair_cut(term_of(a, term), term_of(c, term));
            }
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= alpha;
        if (every) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const u32x4 v = *reinterpret_cast<const u32x4 *>(vp + (int64_t)d * 16 * P);
                o[d] = mma(widen8(v[0], v[1]), pf[0], o[d]);
                o[d] = mma(widen8(v[2], v[3]), pf[1], o[d]);
            }
        } else {
            // Codes that no row sees read as zero.  What some rows see and others do not may be NaN, and a
            // zero weight would not hide it: NaN codes are taken out, counted per row, and put back.
            uint32_t keep[4], seen[4];
            const int hi = in_v ? see_hi : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                keep[i] = byte_mask(tv + 4 * i, see_lo, hi);
                seen[i] = byte_mask(tv + 4 * i, vis_lo, in_v ? vis_hi : 0) & 0x01010101u;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4 v = *reinterpret_cast<const u32x4 *>(vp + (int64_t)d * 16 * P), bad;
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] &= keep[i];
                    bad[i] = nan_bytes(v[i]);
                    v[i] &= ~(bad[i] * 0xffu);
                    any |= bad[i];
                }
                o[d] = mma(widen8(v[0], v[1]), pf[0], o[d]);
                o[d] = mma(widen8(v[2], v[3]), pf[1], o[d]);
                if (__builtin_amdgcn_ballot_w64(any != 0)) {
                    // 0x38 is 1.0: counts of NaN codes that a row sees
                    f32x4 hit = {0, 0, 0, 0};
                    hit = mma(widen8(bad[0] * 0x38u, bad[1] * 0x38u), widen8(seen[0] * 0x38u, seen[1] * 0x38u), hit);
                    hit = mma(widen8(bad[2] * 0x38u, bad[3] * 0x38u), widen8(seen[2] * 0x38u, seen[3] * 0x38u), hit);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] = hit[i] > 0.0f ? NAN : o[d][i];
                }
            }
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

// Joins the token splits of one query row and head.
template <bool BF>
__global__ __launch_bounds__(256) void kv_join_kernel(const KvAttend p, const KvPart part, int splits, int chunk,
                                                      int rows_per_tile, int64_t rows_total) {
    const int b = blockIdx.z, h = blockIdx.y, D = p.c.dim;
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
    float top = -INFINITY;
    for (int s = 0; s < used; ++s) top = fmaxf(top, part.ml[(at + s * step) * 2]);
    const float ref = top == -INFINITY ? 0.0f : top;
    for (int d = threadIdx.x; d < D; d += 256) {
        float val = 0.0f, tot = 0.0f;
        for (int s = 0; s < used; ++s) {
            const float f = __builtin_amdgcn_exp2f(part.ml[(at + s * step) * 2] - ref);
            tot += f * part.ml[(at + s * step) * 2 + 1];
            val += f * part.o[(at + s * step) * D + d];
        }
        const float o = tot == 0.0f ? 0.0f : val / tot;
        const int64_t to = (start + i) * p.out_ld + (int64_t)h * D + d;
        if constexpr (BF) static_cast<__bf16 *>(p.out)[to] = (__bf16)o;
        else static_cast<float *>(p.out)[to] = o;
    }
}

template <bool BF>
hipError_t attend_rows(const KvAttend &p, const KvPlan &pl, void *workspace, hipStream_t stream) {
    const int group = p.q_heads / p.c.heads, R = BF ? 16 : 4;
    const int row_tiles = (p.b.max_new * group + R - 1) / R;
    const int64_t rows_total = (int64_t)p.b.batch * p.b.max_new;
    KvPart part{};
    part.o = static_cast<float *>(workspace);
    part.ml = part.o + (size_t)pl.splits * rows_total * p.q_heads * p.c.dim;
    const dim3 grid((unsigned)(pl.splits * row_tiles), (unsigned)p.c.heads, (unsigned)p.b.batch);
#define DMC_DIM(N) \
    case N: kv_rows_kernel<N, BF><<<grid, dim3(256), 0, stream>>>(p, part, pl.splits, pl.chunk, row_tiles, rows_total); break;
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

hipError_t launch_kv_append(const KvAppend &p, hipStream_t stream) {
    const int slots = (p.b.max_new + p.c.page - 1) / p.c.page + 1;
    const dim3 grid((unsigned)slots, (unsigned)p.c.heads, (unsigned)p.b.batch * 2);
    if (p.bf16) kv_append_kernel<true><<<grid, dim3(256), 0, stream>>>(p);
    else kv_append_kernel<false><<<grid, dim3(256), 0, stream>>>(p);
    return hipGetLastError();
}

KvPlan plan_kv(const KvAttend &p, int num_cus) {
    KvPlan pl{};
    const int group = p.q_heads / p.c.heads, R = p.bf16 ? 16 : 4;
    const int64_t tiles = (int64_t)((p.b.max_new * group + R - 1) / R) * p.c.heads * p.b.batch;
    int64_t span = p.b.max_len;
    if (p.window > 0) span = std::min<int64_t>(span, p.window + R + kStep);
    const int64_t units = std::max<int64_t>(1, (span + 4 * kStep - 1) / (4 * kStep));
    const int64_t want = std::max<int64_t>(1, 4 * num_cus / std::max<int64_t>(1, tiles));
    const int64_t per = (units + want - 1) / want;  // steps of 256 tokens per workgroup
    pl.chunk = (int)(per * 4 * kStep);
    pl.splits = (int)((units + per - 1) / per);
    if (pl.splits > 1)
        pl.workspace_bytes = (size_t)pl.splits * p.b.batch * p.b.max_new * p.q_heads * (p.c.dim + 2) * 4;
    return pl;
}

hipError_t launch_kv_attend(const KvAttend &p, const KvPlan &pl, void *workspace, hipStream_t stream) {
    return p.bf16 ? attend_rows<true>(p, pl, workspace, stream) : attend_rows<false>(p, pl, workspace, stream);
}

}  // namespace dmc
