// Long contexts: rows rotated into a paged cache, the bounds of its blocks, the blocks that a row reads, and attention over them
// (voxhip.h: vox_rope_append, vox_block_bounds, vox_block_select, vox_block_attention).
#include "vox_internal.h"

typedef _Float16 half_t;

// one element of either 16-bit type, as its bits <-> fp32
template <int F16>
__device__ __forceinline__ float elem_f(bf16_t b) {
    if constexpr (F16) { union { uint16_t u; half_t h; } c; c.u = b; return (float)c.h; }
    else return bf2f(b);
}
// (fp16: f is rounded to 32 bits first, as everywhere - left to itself the compiler joins a multiply-add and the conversion to one instruction that rounds
// once, and a value in 20000 comes out one fp16 step from the other order's)
template <int F16>
__device__ __forceinline__ bf16_t f_elem(float f) {
    if constexpr (F16) { asm("" : "+v"(f)); union { uint16_t u; half_t h; } c; c.h = (half_t)f; return c.u; }
    else return f2bf(f);
}

// The step of values whose largest finite magnitude is amax: the smallest power of two of which 127 reach it, at least 2^-100.
__device__ __forceinline__ float step_of(float amax) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 126;        // amax = f 2^e, f in [0.5, 1); (subnormal amax: e = -126, the floor below)
    const int m = e - 7 < -100 ? -100 : e - 7;
    float s = __uint_as_float((u32)(m + 127) << 23);
    if (amax > 127.0f * s) s *= 2.0f;                               // (not at the floor: there 127 s is far above)
    return s;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __uint_as_float(0x7f800000u) ? a : 0.0f;             // NaN and infinities: 0
}

static int check_cache(const char* who, const vox_block_cache& c, bool bounds) {
    if (!c.kv) return vox_fail(VOX_ERR_INVALID, "%s: no cache", who);
    if (c.n_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return vox_fail(VOX_ERR_INVALID, "%s: %d pages of %d tokens, %d kv heads", who, c.n_pages, c.page_size, c.kv_heads);
    if (c.dtype != VOX_DTYPE_BF16 && c.dtype != VOX_DTYPE_F16) return vox_fail(VOX_ERR_INVALID, "%s: dtype %d", who, c.dtype);
    if ((size_t)c.kv & 15) return vox_fail(VOX_ERR_INVALID, "%s: the cache does not lie on 16 bytes", who);
    if (!bounds) return VOX_OK;
    if (c.block != 16 && c.block != 32 && c.block != 64 && c.block != 128) return vox_fail(VOX_ERR_INVALID, "%s: blocks of %d tokens (16, 32, 64 or 128)", who, c.block);
    if (c.page_size % c.block) return vox_fail(VOX_ERR_INVALID, "%s: pages of %d tokens are not whole blocks of %d", who, c.page_size, c.block);
    if (c.head_dim != 64 && c.head_dim != 128) return vox_fail(VOX_ERR_INVALID, "%s: head_dim %d (64 or 128)", who, c.head_dim);
    return VOX_OK;
}
static int check_bounds(const char* who, const vox_block_cache& c) {
    if (!c.bounds || !c.steps) return vox_fail(VOX_ERR_INVALID, "%s: no bounds or no steps", who);
    if ((size_t)c.bounds & 15 || (size_t)c.steps & 3) return vox_fail(VOX_ERR_INVALID, "%s: bounds on 16 bytes, steps on 4", who);
    return VOX_OK;
}
static int check_rows(const char* who, const vox_block_cache& c, const vox_block_rows& r) {
    if (r.n_rows < 0 || r.n_req < 0 || r.n_own < 0 || r.max_kvlen < 0) return vox_fail(VOX_ERR_INVALID, "%s: %d rows of %d requests, max_kvlen %d", who, r.n_rows, r.n_req, r.max_kvlen);
    if (r.heads <= 0 || r.heads % c.kv_heads || r.heads / c.kv_heads > 64) return vox_fail(VOX_ERR_INVALID, "%s: %d heads on %d kv heads (1 to 64 on each)", who, r.heads, c.kv_heads);
    if (r.n_rows && (!r.q_req || !r.q_kvlen || !r.kv_indptr || !r.kv_indices)) return vox_fail(VOX_ERR_INVALID, "%s: a plan array is NULL", who);
    return VOX_OK;
}
template <class A>
static int launch(const void* kern, dim3 grid, int threads, size_t lds, hipStream_t st, A& a) {
    void* args[] = {&a};
    if (lds > 64 * 1024) VOX_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    VOX_HIP(hipLaunchKernel(kern, grid, dim3(threads), args, lds, st));
    return VOX_OK;
}

// ================================================================================================
// rotate and append
// ================================================================================================
struct RopeAppendArgs {
    const bf16_t *q, *k, *v;
    bf16_t *q_out, *kv;
    const int *pos, *page, *slot;
    const float* cs;
    int8_t* bounds;                      // blocks of threads from `append_blocks` on: the bounds of the blocks that the rows complete
    float* steps;
    long q_stride, k_stride, v_stride;
    int n_rows, Hq, Hkv, D, rot, interleave, max_pos, page_size, n_pages, block, slots, append_blocks;
};
__device__ __forceinline__ bool row_place(const int* page, const int* slot, int n, int n_pages, int page_size, int& pg, int& sl) {
    pg = page[n]; sl = slot[n];
    return pg >= 0 && pg < n_pages && sl >= 0 && sl < page_size;
}
__device__ __forceinline__ int table_row(const RopeAppendArgs& a, int n) {
    const int p = a.rot ? a.pos[n] : 0;
    return p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
}
template <int F16>
__device__ __forceinline__ void turn(float x, float y, float c, float s, bf16_t& u, bf16_t& v) {
    u = f_elem<F16>(__fmaf_rn(-y, s, x * c));
    v = f_elem<F16>(__fmaf_rn(x, s, y * c));
}

// Any dims, strides and alignment: one thread a pair of channels that turn together (or two that do not).
template <int F16>
__global__ __launch_bounds__(256) void k_rope_append_any(RopeAppendArgs a) {
    const int half_d = a.D >> 1, half = a.rot >> 1, pairs = (a.Hq + 2 * a.Hkv) * half_d;
    const long item = (long)blockIdx.x * 256 + threadIdx.x;
    const int n = (int)(item / pairs), i = (int)(item % pairs);
    int pg, slot;
    if (n >= a.n_rows || !row_place(a.page, a.slot, n, a.n_pages, a.page_size, pg, slot)) return;
    const int p = table_row(a, n), head = i / half_d, c = i % half_d;
    const int kind = head < a.Hq ? 0 : head < a.Hq + a.Hkv ? 1 : 2, h = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - a.Hkv;
    const bf16_t* const src = (kind == 0 ? a.q + n * a.q_stride : kind == 1 ? a.k + n * a.k_stride : a.v + n * a.v_stride) + (size_t)h * a.D;
    bf16_t* const dst = kind == 0 ? a.q_out + ((size_t)n * a.Hq + h) * a.D
                                  : a.kv + (((size_t)pg * 2 + (kind == 2)) * a.page_size + slot) * a.Hkv * a.D + (size_t)h * a.D;
    const bool turns = kind < 2 && c < half;
    const int i0 = turns && !a.interleave ? c : turns || kind == 2 ? 2 * c : a.rot + 2 * (c - half), i1 = turns && !a.interleave ? c + half : i0 + 1;
    bf16_t x = src[i0], y = src[i1];
    if (turns) turn<F16>(elem_f<F16>(x), elem_f<F16>(y), a.cs[((size_t)p * half + c) * 2], a.cs[((size_t)p * half + c) * 2 + 1], x, y);
    dst[i0] = x;
    dst[i1] = y;
}

// The bounds of one block, by one wave: D / 8 lanes hold a key, 512 / D keys at once.  key(l, t): channels 8 l .. 8 l + 7 of token t.
template <int F16, int D, class K>
__device__ __forceinline__ void block_bounds(int lane, int block, int8_t* bounds, float* step_out, K key) {
    constexpr int LPT = D / 8, TPI = 64 / LPT;
    const float inf = __uint_as_float(0x7f800000u);
    const int l = lane % LPT;
    float hi[8], lo[8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) { hi[i] = -inf; lo[i] = inf; }
#pragma unroll 4
    for (int t = lane / LPT; t < block; t += TPI) {
        const uint4 v = key(l, t);
        const u32 w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = elem_f<F16>((bf16_t)(w[i / 2] >> (16 * (i % 2))));
            hi[i] = x > hi[i] ? x : hi[i];                          // (false for NaN)
            lo[i] = x < lo[i] ? x : lo[i];
            amax = fmaxf(amax, finite_abs(x));                      // (of all keys: infinities would stand in front of it in the bounds)
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int o = LPT; o < 64; o <<= 1) {
            hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], o, 64));
            lo[i] = fminf(lo[i], __shfl_xor(lo[i], o, 64));
        }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    const float step = step_of(amax), inv = 1.0f / step;
    if (lane < LPT) {
        u32 wh[2] = {0, 0}, wl[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool any = hi[i] >= lo[i];                        // (a channel of NaN: no)
            const int H = any ? (int)fminf(fmaxf(ceilf(hi[i] * inv), -127.0f), 127.0f) : 0, L = any ? (int)fminf(fmaxf(floorf(lo[i] * inv), -127.0f), 127.0f) : 0;
            wh[i / 4] |= (u32)(H & 255) << (8 * (i % 4));
            wl[i / 4] |= (u32)(L & 255) << (8 * (i % 4));
        }
        *reinterpret_cast<uint2*>(bounds + 8 * l) = make_uint2(wh[0], wh[1]);
        *reinterpret_cast<uint2*>(bounds + D + 8 * l) = make_uint2(wl[0], wl[1]);
        if (lane == 0) *step_out = step;
    }
}

// Vectors: a thread has 16 channels of a head that turn (two runs of eight whose pairs they are: halves, or 16 in a row: neighbours) or do not, and goes through the
// row's heads slot, slot + slots, ..: the angles are loaded once.  Calls of few rows take a slot a head (everything in flight at once), calls of many rows eight
// slots a row (the angles, 64 bytes a thread, would be as much to load as the channels).
// With rows of different requests the launch has more blocks of threads behind these: a wave a row and kv head, which leaves at once unless the row
// completes a block; the other keys of the block are in the cache from earlier calls, the row's own is turned here once more.
template <int F16, int IL, int D>        // D: 64 or 128 with bounds, else 0 (any)
__global__ __launch_bounds__(256) void k_rope_append(RopeAppendArgs a) {
    if constexpr (D > 0) if ((int)blockIdx.x >= a.append_blocks) {
        const int at = ((int)blockIdx.x - a.append_blocks) * 4 + (threadIdx.x >> 6), n = at / a.Hkv, h = at % a.Hkv, half = a.rot >> 1;
        int pg, slot;
        if (n >= a.n_rows || !row_place(a.page, a.slot, n, a.n_pages, a.page_size, pg, slot) || (slot + 1) % a.block) return;
        const int p = table_row(a, n), per = a.page_size / a.block;
        const bf16_t* const base = a.kv + ((size_t)pg * 2 * a.page_size + slot + 1 - a.block) * a.Hkv * D + (size_t)h * D;
        const bf16_t* const own = a.k + n * a.k_stride + (size_t)h * D;
        const size_t to = ((size_t)pg * a.Hkv + h) * per + slot / a.block;
        block_bounds<F16, D>(threadIdx.x & 63, a.block, a.bounds + to * 2 * D, a.steps + to, [&](int l, int t) {
            if (t + 1 < a.block) return *reinterpret_cast<const uint4*>(base + (size_t)t * a.Hkv * D + 8 * l);
            bf16_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int ch = 8 * l + i;
                e[i] = own[ch];
                if (ch < a.rot) {
                    const int pair = IL ? ch >> 1 : ch % half;
                    const bool second = IL ? ch & 1 : ch >= half;
                    const float other = elem_f<F16>(own[IL ? ch ^ 1 : second ? ch - half : ch + half]), me = elem_f<F16>(e[i]);
                    bf16_t u, v;
                    turn<F16>(second ? other : me, second ? me : other, a.cs[((size_t)p * half + pair) * 2], a.cs[((size_t)p * half + pair) * 2 + 1], u, v);
                    e[i] = second ? v : u;
                }
            }
            return make_uint4((u32)e[0] | ((u32)e[1] << 16), (u32)e[2] | ((u32)e[3] << 16), (u32)e[4] | ((u32)e[5] << 16), (u32)e[6] | ((u32)e[7] << 16));
        });
        return;
    }
    const int units = a.D >> 4, per_row = units * a.slots, heads = a.Hq + 2 * a.Hkv;
    const long item = (long)blockIdx.x * 256 + threadIdx.x;
    const int n = (int)(item / per_row), j = (int)(item - (long)n * per_row), u = j % units, slot0 = j / units;
    int pg, slot;
    if (n >= a.n_rows || !row_place(a.page, a.slot, n, a.n_pages, a.page_size, pg, slot)) return;
    const int half = a.rot >> 1;
    const bool turns = 16 * u < a.rot;
    const int c0 = turns && !IL ? 8 * u : 16 * u, c1 = turns && !IL ? half + 8 * u : c0 + 8;
    float cs[16];
    if (turns) {
        const float4* const t = reinterpret_cast<const float4*>(a.cs + ((size_t)table_row(a, n) * half + 8 * u) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 x = t[i];
            cs[4 * i] = x.x; cs[4 * i + 1] = x.y; cs[4 * i + 2] = x.z; cs[4 * i + 3] = x.w;
        }
    }
    bf16_t* const kd = a.kv + ((size_t)pg * 2 * a.page_size + slot) * a.Hkv * a.D;
    auto from = [&](int head) { return head < a.Hq ? a.q + n * a.q_stride + (size_t)head * a.D
                                     : head < a.Hq + a.Hkv ? a.k + n * a.k_stride + (size_t)(head - a.Hq) * a.D : a.v + n * a.v_stride + (size_t)(head - a.Hq - a.Hkv) * a.D; };
    constexpr int B = 3;                                             // heads in flight
    for (int h0 = slot0; h0 < heads; h0 += B * a.slots) {
        uint4 x[B], y[B];
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (h0 + b * a.slots < heads) {
                const bf16_t* const src = from(h0 + b * a.slots);
                x[b] = *reinterpret_cast<const uint4*>(src + c0);
                y[b] = *reinterpret_cast<const uint4*>(src + c1);
            }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int head = h0 + b * a.slots;
            if (head >= heads) break;
            bf16_t* const dst = head < a.Hq ? a.q_out + ((size_t)n * a.Hq + head) * a.D
                              : head < a.Hq + a.Hkv ? kd + (size_t)(head - a.Hq) * a.D : kd + ((size_t)a.page_size * a.Hkv + head - a.Hq - a.Hkv) * a.D;
            if (turns && head < a.Hq + a.Hkv) {
                u32 w[8] = {x[b].x, x[b].y, x[b].z, x[b].w, y[b].x, y[b].y, y[b].z, y[b].w};
                bf16_t e[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) e[i] = (bf16_t)(w[i / 2] >> (16 * (i % 2)));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    bf16_t& s = e[IL ? 2 * i : i];
                    bf16_t& t = e[IL ? 2 * i + 1 : 8 + i];
                    turn<F16>(elem_f<F16>(s), elem_f<F16>(t), cs[2 * i], cs[2 * i + 1], s, t);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = (u32)e[2 * i] | ((u32)e[2 * i + 1] << 16);
                x[b] = make_uint4(w[0], w[1], w[2], w[3]);
                y[b] = make_uint4(w[4], w[5], w[6], w[7]);
            }
            *reinterpret_cast<uint4*>(dst + c0) = x[b];
            *reinterpret_cast<uint4*>(dst + c1) = y[b];
        }
    }
}

struct BoundsArgs {
    const bf16_t* kv;
    int8_t* bounds;
    float* steps;
    const int *page, *slot;
    int n_rows, n_pages, page_size, block, Hkv;
};
// 64 rows and a kv head a block of threads; its waves share the rows that complete a block
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_bounds(BoundsArgs a) {
    const int n0 = blockIdx.x * 64, h = blockIdx.y, lane = threadIdx.x & 63;
    int pg = -1, slot = 0;
    const bool done = n0 + lane < a.n_rows && row_place(a.page, a.slot, n0 + lane, a.n_pages, a.page_size, pg, slot) && (slot + 1) % a.block == 0;
    unsigned long long left = __ballot(done);
    for (int i = 0; left; ++i, left &= left - 1) {
        if ((i & 3) != (int)(threadIdx.x >> 6)) continue;
        const int from = __builtin_ctzll(left), p = __shfl(pg, from, 64), s = __shfl(slot, from, 64);
        const bf16_t* const k = a.kv + ((size_t)p * 2 * a.page_size + s + 1 - a.block) * a.Hkv * D + (size_t)h * D;
        const size_t to = ((size_t)p * a.Hkv + h) * (a.page_size / a.block) + s / a.block;
        block_bounds<F16, D>(lane, a.block, a.bounds + to * 2 * D, a.steps + to, [&](int l, int t) { return *reinterpret_cast<const uint4*>(k + (size_t)t * a.Hkv * D + 8 * l); });
    }
}

// ================================================================================================
// choose
// ================================================================================================
struct SelectArgs {
    const bf16_t* q;
    const int8_t* bounds;
    const float* steps;
    const int *q_req, *q_kvlen, *indptr, *indices;
    int* blocks;
    long q_stride;
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top, first, last, stride;
};
// order of the scores as unsigned numbers; 0 is below all of them
__device__ __forceinline__ u32 score_key(float s) {
    const u32 b = __float_as_uint(s);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ int q_steps(float x, float inv) {
    const float t = fminf(fmaxf(__builtin_rintf(x * inv), -127.0f), 127.0f);
    return x == x ? (int)t : 0;
}
typedef int i32x4 __attribute__((ext_vector_type(4)));

// The scores of QT rows of one request (or of one row) and a kv head, then their choice.
//   sum over heads and channels of max(a hi, a lo) = sum over channels of P hi + N lo, P = sum over heads of max(a, 0), N of min(a, 0): one product of 2 dim
// whole numbers however many heads there are.  P and N have up to 13 bits; 64 times their high part and their low six bits are two rows of an 8-bit matrix
// product, so 16 rows of it are 8 query rows, and 16 blocks its columns: C's lanes have both rows of a query beside each other.
// A tile of 16 (or 8) query rows reads the bounds of a request's blocks once; what a choice costs is its rounds over the keys, in a wave's registers.
// The keys of all candidates lie in LDS: [row][SEL_STRIDE(blocks)].
#define SEL_PAD 8
// keys of one row, a wave's or W waves' (W > 1: all threads call): the need largest, older first where equal, written in order of their index
template <int KPL, int W>
__device__ __forceinline__ void choose(const u32* key, int lo, int cand, int need, int first, int last, int have, int top, int* out, int lane, int wave, int (*red)[16]) {
    u32 k[KPL];
    const int c0 = W > 1 ? wave * KPL * 64 : 0;
    u32 least = 0xffffffffu, most = 0;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        const int c = c0 + i * 64 + lane;
        const bool in = c < cand;
        k[i] = in ? key[lo + c] : 0;                                 // (0: below every key but that of a block without a page, and counted with care)
        least = min(least, in ? k[i] : 0xffffffffu);
        most = max(most, k[i]);
    }
    int turn_ = 0;
    auto total = [&](int x) {                                        // over the row's waves
        if constexpr (W > 1) {
            int* const r = red[turn_ & 1];
            ++turn_;
            if (lane == 0) r[wave] = x;
            __syncthreads();
            x = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) x += r[w];
        }
        return x;
    };
    // the need-th largest key t lies in [a, b): at least need keys reach a, fewer reach b
    for (int o = 1; o < 64; o <<= 1) {
        least = min(least, (u32)__shfl_xor((int)least, o, 64));
        most = max(most, (u32)__shfl_xor((int)most, o, 64));
    }
    if constexpr (W > 1) {
        u32* const r = reinterpret_cast<u32*>(red[2]);
        u32* const s = reinterpret_cast<u32*>(red[3]);
        if (lane == 0) { r[wave] = least; s[wave] = most; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) { least = min(least, r[w]); most = max(most, s[w]); }
    }
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
    u32 a = least, t = least, above = 0;
    unsigned long long b = (unsigned long long)most + 1;
    bool exact = false;                                              // exactly `need` keys reach t: no ties to break
    if (need == 0) { t = 0xffffffffu; exact = true; }
    while (!exact && b - a > 1) {
        const u32 mid = a + (u32)((b - a) >> 1);
        int n = 0;
#pragma unroll
        for (int i = 0; i < KPL; ++i) n += (int)__popcll(__ballot(k[i] >= mid));      // (mid > least >= 0: lanes outside, 0, never reach it)
        n = total(n);
        if (n >= need) a = mid; else b = mid;
        if (n == need) { exact = true; }
        t = a;
    }
    (void)above;
    // keys above t, and the oldest equal ones
    int gt = 0, eq = 0;
    if (need && !exact) {
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const bool in = c0 + i * 64 + lane < cand;
            gt += (int)__popcll(__ballot(in && k[i] > t));
            eq += (int)__popcll(__ballot(in && k[i] == t));
        }
    } else if (need) {
#pragma unroll
        for (int i = 0; i < KPL; ++i) gt += (int)__popcll(__ballot(c0 + i * 64 + lane < cand && k[i] >= t));
    }
    int gt_before = 0, eq_before = 0, gt_all = gt;
    if constexpr (W > 1) {
        __syncthreads();
        if (lane == 0) { red[0][wave] = gt; red[1][wave] = eq; }
        __syncthreads();
        gt_all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < wave) { gt_before += red[0][w]; eq_before += red[1][w]; }
            gt_all += red[0][w];
        }
    }
    int ties = exact ? 0 : need - gt_all;                            // equal ones to take, from the oldest
    const unsigned long long below = lane ? ~0ull >> (64 - lane) : 0ull;
    int at = first + gt_before + min(eq_before, ties);
    ties = max(ties - eq_before, 0);
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        if (c0 + i * 64 >= cand || need == 0) break;
        const bool in = c0 + i * 64 + lane < cand, e = in && !exact && k[i] == t, g = in && (exact ? k[i] >= t : k[i] > t);
        const unsigned long long be = __ballot(e);
        const bool take = g || (e && (int)__popcll(be & below) < ties);
        const unsigned long long bt = __ballot(take);
        if (take) out[at + (int)__popcll(bt & below)] = lo + c0 + i * 64 + lane;
        at += (int)__popcll(bt);
        ties -= min(ties, (int)__popcll(be));
    }
    if (W == 1 || wave == 0) {
        for (int j = lane; j < first; j += 64) out[j] = j;
        for (int j = lane; j < last; j += 64) out[top - last + j] = have - last + j;
    }
}

// QT > 1: tiles of QT rows, a wave a row in the choice; QT == 1: a row, all waves together
template <int F16, int D, int QT, int W>
__global__ __launch_bounds__(64 * W) void k_block_select(SelectArgs a) {
    constexpr int MT = (2 * QT + 15) / 16, KS = 2 * D / 64;          // tiles of 16 product rows, steps of 64 numbers
    extern __shared__ __attribute__((aligned(16))) u32 keys[];       // [QT][a.stride]
    __shared__ __attribute__((aligned(16))) int8_t s_a[MT * 16][2 * D];
    __shared__ int s_len[QT], s_req[QT], red[4][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int h = blockIdx.x % a.Hkv, i0 = blockIdx.x / a.Hkv * QT, R = min(QT, a.n_rows - i0), G = a.Hq / a.Hkv, per = a.page_size / a.block;
    if (tid < QT) {
        int n = 0, r = -1;
        if (tid < R) {
            n = a.q_kvlen[i0 + tid];
            r = a.q_req[i0 + tid];
            if (n <= 0 || r < 0 || r >= a.n_req) { n = 0; r = -1; }
            n = min(n, a.max_kvlen);
            if (n == 0) r = -1;
        }
        s_len[tid] = n; s_req[tid] = r;
    }
    if constexpr (QT < 8) for (int x = tid; x < (MT * 16 - 2 * QT) * 2 * D / 4; x += 64 * W) reinterpret_cast<int*>(s_a[2 * QT])[x] = 0;
    // P and N of the rows, a wave a row
    for (int r = wave; r < R; r += W) {
        const bf16_t* const q = a.q + (size_t)(i0 + r) * a.q_stride + (size_t)h * G * D;
        float amax = 0.0f;
        for (int e = lane; e < G * D; e += 64) amax = fmaxf(amax, finite_abs(elem_f<F16>(q[e])));
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
        const float inv = 1.0f / step_of(amax);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            const int d = lane + 64 * x;
            int p = 0, m = 0;
            for (int e = 0; e < G; ++e) {
                const int s = q_steps(elem_f<F16>(q[e * D + d]), inv);
                p += max(s, 0); m += min(s, 0);
            }
            s_a[2 * r][d] = (int8_t)(p & 63); s_a[2 * r + 1][d] = (int8_t)(p >> 6);
            s_a[2 * r][D + d] = (int8_t)(m & 63); s_a[2 * r + 1][D + d] = (int8_t)(m >> 6);
        }
    }
    __syncthreads();
    i32x4 av[MT][KS];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < KS; ++s) av[t][s] = *reinterpret_cast<const i32x4*>(&s_a[16 * t + c][64 * s + 16 * g]);

    for (int ra = 0; ra < R;) {
        if (s_req[ra] < 0) { ++ra; continue; }
        int rb = ra + 1;
        while (rb < R && s_req[rb] == s_req[ra]) ++rb;
        const int req = s_req[ra], p0 = a.indptr[req], np = a.indptr[req + 1] - p0;
        int n_most = 0;
        for (int r = ra; r < rb; ++r) n_most = max(n_most, s_len[r]);
        const int have = (n_most + a.block - 1) / a.block, j1 = have > a.top ? have - a.last : 0;      // blocks to score: [first, j1)
        constexpr int U = 4;                                         // tiles of 16 blocks in flight
        for (int j0 = a.first + wave * 16 * U; j0 < j1; j0 += W * 16 * U) {
            int pg[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + 16 * u + c, pj = j / per;
                pg[u] = j < j1 && pj < np ? a.indices[p0 + pj] : -1;
            }
            i32x4 b[U][KS];
            float st[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + 16 * u + c;
                const bool ok = pg[u] >= 0 && pg[u] < a.n_pages;
                const size_t at = ok ? ((size_t)pg[u] * a.Hkv + h) * per + j % per : 0;
                const i32x4* const src = reinterpret_cast<const i32x4*>(a.bounds + at * 2 * D) + g;
#pragma unroll
                for (int s = 0; s < KS; ++s) b[u][s] = src[4 * s];
                st[u] = a.steps[at];
                pg[u] = ok;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = j0 + 16 * u + c;
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    i32x4 s4 = {0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < KS; ++s) s4 = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[t][s], b[u][s], s4, 0, 0, 0);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {                    // product rows 4 g + 2 x, + 1: query row 8 t + 2 g + x
                        const int r = 8 * t + 2 * g + x;
                        if (j < j1 && r < QT) keys[(size_t)r * a.stride + j] = pg[u] ? score_key((float)(s4[2 * x] + 64 * s4[2 * x + 1]) * st[u]) : 0;
                    }
                }
            }
        }
        __syncthreads();
        for (int r = ra + (QT > 1 ? wave : 0); r < rb; r += QT > 1 ? W : 1) {
            const int mine = (s_len[r] + a.block - 1) / a.block, cand = mine - a.first - a.last, need = a.top - a.first - a.last;
            int* const out = a.blocks + ((size_t)(i0 + r) * a.Hkv + h) * a.top;
            if (mine <= a.top) {
                for (int j = QT > 1 ? lane : tid; j < a.top; j += QT > 1 ? 64 : 64 * W) out[j] = j < mine ? j : -1;
                continue;
            }
            const u32* const key = keys + (size_t)r * a.stride;
            constexpr int GW = QT > 1 ? 1 : W;
#define CHOOSE(KPL) choose<KPL, GW>(key, a.first, cand, need, a.first, a.last, mine, a.top, out, lane, wave, red)
            if (cand <= 4 * 64 * GW) CHOOSE(4);
            else if (cand <= 8 * 64 * GW) CHOOSE(8);
            else if (cand <= 16 * 64 * GW) CHOOSE(16);
            else if constexpr (QT == 1 || QT == 8) { if (cand <= 32 * 64 * GW) CHOOSE(32); else CHOOSE(64); }
#undef CHOOSE
        }
        __syncthreads();
        ra = rb;
    }
}

// ================================================================================================
// attend
// ================================================================================================
// Sixteen columns - the query heads of one kv head (up to 16 of them), of one row or of as many neighbouring rows of a request as fit - meet the blocks that
// any of their rows lists, 32 tokens at a time: two tiles of 16, of one block or of two.
//   S^T = K Q^T     A: a token a lane, 8 channels; lane (c, g) then holds the scores of column c = lane % 16 for tokens 4 g .. 4 g + 3 (g = lane / 16) of each tile,
//   O^T = V^T P^T   B: these same scores' weights, where they are - the order of the 32 tokens inside a product is free, so V's lanes take tokens 4 g ..
//                   4 g + 3 of each tile too.  A lane loads 8 neighbouring channels (D = 128) of its 8 tokens, whole rows a sixteen lanes, and a tile t of
//                   the product takes channel 8 m + t of each: halves of registers by v_perm, no LDS.
// Maximum and sum of a column stay with its lanes (online softmax, exponents of two, fp32).  A weight enters as the sum of two 16-bit terms: one alone would
// cost as much precision as the output's own rounding.
// What a column must not see is kept from it by its score alone (weight 0), which holds as long as V is finite; where a result is not, the rows are gone through
// again one by one in the same order with V's masked tokens as zero, and a value that is not finite multiplied by the weight as one term (an infinity times the
// two terms would be inf - inf).  Rows that see no such value come out bit for bit as if it were not there.
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef half_t f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int F16>
__device__ __forceinline__ f32x4 mma32(uint4 a, uint4 b, f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int F16>
__device__ __forceinline__ u32 pack2(float lo, float hi) {
    if constexpr (F16) return (u32)f_elem<1>(lo) | ((u32)f_elem<1>(hi) << 16);
    else return pack_bf2(lo, hi);
}
template <int OFF>                       // 16 or 32
__device__ __forceinline__ float xor_max(float s) {
    vox_u2 r;
    if constexpr (OFF == 32) r = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    else r = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
template <int F16>
__device__ __forceinline__ u32 halves_not_finite(u32 w) {          // 0xffff where a half is an infinity or NaN
    const u32 e = F16 ? 0x7c00u : 0x7f80u;
    return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}

struct BlockAttnArgs {
    const bf16_t *q, *kv;
    const int *q_req, *q_kvlen, *indptr, *indices, *blocks;
    bf16_t* out;
    float *part_o, *part_ml;             // splits > 1: [row][head][split][D], [row][head][split][2]
    long q_stride;
    float scale2;                        // scale log2 e
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top;
    int per_tile, splits, head_tiles, cols, q_al, out_al;      // cols: columns of a wave in the merge's LDS
};
#define ATTN_CUS 256                     // of an MI355X
#define ATTN_WINDOW 4096                 // blocks whose rows' bits lie in LDS at a time (rows of several: 8 KB)

// The entries of a row's list that count, 64 at a time, by one wave: f(j, counts) for every lane.
template <class F>
__device__ __forceinline__ void row_entries(const int* list, int top, int have, int lane, F f) {
    int carry = -1;
    for (int e0 = 0; e0 < top; e0 += 64) {
        const int j = e0 + lane < top ? list[e0 + lane] : -1;
        int most = j;                                                // the largest entry up to this one
        const int prev = __shfl_up(j, 1, 64);
        if (__ballot(lane && j >= 0 && j <= prev) || __ballot(lane && j >= 0 && prev < 0))      // (not simply ascending)
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(most, o, 64);
                if (lane >= o) most = max(most, x);
            }
        int before = __shfl_up(most, 1, 64);
        before = lane ? max(before, carry) : carry;
        f(j, j >= 0 && j > before && j < have);
        if (e0 + 64 < top) {                                         // the carry of the next 64
            int last = j;
            for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o, 64));
            carry = max(carry, last);
        }
    }
}

template <int F16, int D, int W, bool ONE>
__global__ __launch_bounds__(64 * W, W == 4 ? 2 : 1) void k_block_attn(BlockAttnArgs a) {
    constexpr int CPL = D / 16, KS = D / 32, OS = D + 4;             // channels a lane, steps of a K row, floats a column of the merge
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int s_len[16], s_req[16], s_count[W + 1], s_next, s_seen;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const float inf = __uint_as_float(0x7f800000u);
    // block -> (kv head, tile of heads, split, tile of rows): neighbours are kv heads, so that a die's L2 keeps its heads' tokens
    int id = blockIdx.x;
    const int h = id % a.Hkv; id /= a.Hkv;
    const int ht = id % a.head_tiles; id /= a.head_tiles;
    const int split = id % a.splits, tile = id / a.splits;
    const int G = a.Hq / a.Hkv, h0 = ht * 16, gh = min(G - h0, 16);  // this tile's heads
    const int i0 = tile * a.per_tile, R = min(a.per_tile, a.n_rows - i0);
    if (tid < 16) {
        int len = 0, req = -1;
        if (tid < R) {
            len = a.q_kvlen[i0 + tid];
            req = a.q_req[i0 + tid];
            if (len <= 0 || req < 0 || req >= a.n_req) { len = 0; req = -1; }
            len = min(len, a.max_kvlen);
        }
        s_len[tid] = len; s_req[tid] = req;
    }
    __syncthreads();
    const int rc = ONE ? 0 : c / gh, hc = ONE ? c : c % gh;          // the column's row and head
    const bool col = ONE ? c < gh : rc < R;
    uint4 q[KS];
    {
        const bf16_t* const src = a.q + (size_t)(i0 + (col ? rc : 0)) * a.q_stride + (size_t)(h * G + h0 + (col ? hc : 0)) * D + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (a.q_al) q[s] = *reinterpret_cast<const uint4*>(src + 32 * s);
            else {
                u32 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (u32)src[32 * s + 2 * i] | ((u32)src[32 * s + 2 * i + 1] << 16);
                q[s] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (!col) q[s] = make_uint4(0, 0, 0, 0);
        }
    }
    const int sub_shift = a.block == 16 ? 0 : a.block == 32 ? 1 : a.block == 64 ? 2 : 3, per = a.page_size / a.block;
    const size_t row_el = (size_t)a.Hkv * D;                         // elements between tokens
    int2* const s_list = reinterpret_cast<int2*>(lds);               // {block (from the window's first) << 16 | rows, or the block (ONE); page}
    u32* const s_bits = reinterpret_cast<u32*>(lds);                 // rows of several: two blocks' rows a word, in front of the list
    int2* const list = ONE ? s_list : s_list + ATTN_WINDOW / 4;
    float* const s_o = reinterpret_cast<float*>(lds);                // after the loop: [wave][column][OS]
    float* const s_ml = s_o + W * a.cols * OS;                           // [wave][column] maximum, sum

    for (int ra = 0; ra < R;) {
        if (s_req[ra] < 0) { ++ra; continue; }                       // (all of the block's threads read the same LDS words)
        int rb = ra + 1;
        while (rb < R && s_req[rb] == s_req[ra]) ++rb;
        const int req = s_req[ra], p0 = a.indptr[req], np = a.indptr[req + 1] - p0;
        int n_most = 0, n_least = 0x7fffffff;
        for (int r = ra; r < rb; ++r) { n_most = max(n_most, s_len[r]); n_least = min(n_least, s_len[r]); }
        const u32 all_rows = (rb == 32 ? 0u : 1u << rb) - (1u << ra);
        const int own = ONE ? s_len[ra] : col && rc >= ra && rc < rb ? s_len[rc] : 0;

        for (int careful = -1;;) {                                   // -1, then, if need be, the run's rows one by one
            float m = -inf, l = 0.0f;
            f32x4 o[CPL];
#pragma unroll
            for (int t = 0; t < CPL; ++t) o[t] = f32x4{0, 0, 0, 0};
            const int v_len = careful >= 0 ? s_len[careful] : n_most;     // V of tokens from here on is taken as zero
            if (tid == 0) s_seen = 0;
            __syncthreads();

            for (int w0 = 0; w0 >= 0;) {                             // windows of blocks (ONE: one, of everything)
                int count;
                if constexpr (ONE) {
                    if (wave == 0) {
                        int at = 0;
                        row_entries(a.blocks + ((size_t)i0 * a.Hkv + h) * a.top, a.top, (n_most + a.block - 1) / a.block, lane, [&](int j, bool ok) {
                            int pg = -1;
                            if (ok && j / per < np) pg = a.indices[p0 + j / per];
                            ok = pg >= 0 && pg < a.n_pages;
                            const unsigned long long b = __ballot(ok);
                            if (ok) list[at + __popcll(b & ((1ull << lane) - 1))] = make_int2(j, pg);
                            at += __popcll(b);
                        });
                        if (lane == 0) s_count[0] = at;
                    }
                    __syncthreads();
                    count = s_count[0];
                    if (tid == 0 && count) s_seen = 1;
                    w0 = -1;
                } else {
                    for (int i = tid; i < ATTN_WINDOW / 2; i += 64 * W) s_bits[i] = 0;
                    if (tid == 0) s_next = 0x7fffffff;
                    __syncthreads();
                    for (int r = ra + wave; r < rb; r += W)
                        row_entries(a.blocks + ((size_t)(i0 + r) * a.Hkv + h) * a.top, a.top, (s_len[r] + a.block - 1) / a.block, lane, [&](int j, bool ok) {
                            if (!ok || j < w0) return;
                            if (j - w0 < ATTN_WINDOW) atomicOr(&s_bits[(j - w0) >> 1], 1u << (r + 16 * ((j - w0) & 1)));
                            else atomicMin(&s_next, j);
                        });
                    __syncthreads();
                    // the window's blocks in order: a thread counts its neighbours' share
                    constexpr int WPT = ATTN_WINDOW / 2 / (64 * W);
                    u32 bits[WPT];
                    int mine = 0;
#pragma unroll
                    for (int i = 0; i < WPT; ++i) {
                        bits[i] = s_bits[tid * WPT + i];
                        mine += (bits[i] & 0xffffu ? 1 : 0) + (bits[i] >> 16 ? 1 : 0);
                    }
                    int upto = mine;
                    for (int x = 1; x < 64; x <<= 1) {
                        const int y = __shfl_up(upto, x, 64);
                        if (lane >= x) upto += y;
                    }
                    if (lane == 63) s_count[wave] = upto;
                    __syncthreads();
                    int at = upto - mine;
                    count = 0;
                    for (int x = 0; x < W; ++x) { if (x < wave) at += s_count[x]; count += s_count[x]; }
                    u32 seen = 0;
#pragma unroll
                    for (int i = 0; i < WPT; ++i)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            u32 rows = half ? bits[i] >> 16 : bits[i] & 0xffffu;
                            if (!rows) continue;
                            const int off = (tid * WPT + i) * 2 + half, j = w0 + off;
                            int pg = j / per < np ? a.indices[p0 + j / per] : -1;
                            if (pg < 0 || pg >= a.n_pages) { pg = 0; rows = 0; }      // (nobody's: page 0 is read and masked)
                            list[at++] = make_int2((int)((u32)off << 16 | rows), pg);
                            seen |= rows;
                        }
                    if (seen) atomicOr(&s_seen, (int)seen);
                    __syncthreads();
                }
                const int units = ((count << sub_shift) + 1) / 2;
                const int u0 = ONE ? (int)((long)units * split / a.splits) : 0, u1 = ONE ? (int)((long)units * (split + 1) / a.splits) : units;
                for (int u = u0 + wave; u < u1; u += W) {
                    // two tiles of 16 tokens
                    uint4 k[2][KS];
                    u32 v[2][4][CPL / 2];
                    int tok[2];
                    u32 rows[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int sub = 2 * u + x, e = min(sub >> sub_shift, count - 1), part = sub & ((1 << sub_shift) - 1);
                        const int2 ent = list[e];
                        const int j = ONE ? ent.x : w0 + (int)((u32)ent.x >> 16);
                        rows[x] = (sub >> sub_shift) < count ? (ONE ? 1u : (u32)ent.x & 0xffffu) : 0u;      // (the odd last tile of blocks of 16: nobody's)
                        tok[x] = j * a.block + 16 * part;
                        const bf16_t* const kb = a.kv + ((size_t)ent.y * 2 * a.page_size + (size_t)(j % per) * a.block + 16 * part) * row_el + (size_t)h * D;
                        const bf16_t* const vb = kb + (size_t)a.page_size * row_el;
#pragma unroll
                        for (int s = 0; s < KS; ++s) k[x][s] = *reinterpret_cast<const uint4*>(kb + (size_t)c * row_el + 32 * s + 8 * g);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bf16_t* const src = vb + (size_t)(4 * g + i) * row_el + CPL * c;
                            if constexpr (CPL == 8) {
                                const uint4 t = *reinterpret_cast<const uint4*>(src);
                                v[x][i][0] = t.x; v[x][i][1] = t.y; v[x][i][2] = t.z; v[x][i][3] = t.w;
                            } else {
                                const uint2 t = *reinterpret_cast<const uint2*>(src);
                                v[x][i][0] = t.x; v[x][i][1] = t.y;
                            }
                        }
                    }
                    float p[8];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        f32x4 s4 = {0, 0, 0, 0};
#pragma unroll
                        for (int s = 0; s < KS; ++s) s4 = mma32<F16>(k[x][s], q[s], s4);
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[4 * x + i] = s4[i] * a.scale2;
                        const bool whole = (ONE ? rows[x] != 0 : rows[x] == all_rows) && tok[x] + 16 <= n_least;
                        if (!whole) {
                            const bool mine = ONE ? rows[x] != 0 : (rows[x] >> rc & 1) != 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) p[4 * x + i] = mine && tok[x] + 4 * g + i < own ? p[4 * x + i] : -inf;
                        }
                        // (wave-uniform) V that nobody, or not the careful row, may see
                        const bool none = rows[x] == 0 || (careful >= 0 && !ONE && !(rows[x] >> careful & 1));
                        if (none || tok[x] + 16 > v_len) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const bool drop = none || tok[x] + 4 * g + i >= v_len;
#pragma unroll
                                for (int w = 0; w < CPL / 2; ++w) v[x][i][w] = drop ? 0u : v[x][i][w];
                            }
                        }
                    }
                    float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
                    top = xor_max<32>(xor_max<16>(top));
                    if (__ballot(top > m)) {
                        const float now = fmaxf(m, top), keep = __builtin_amdgcn_exp2f(m - (now == -inf ? 0.0f : now));
                        m = now;
                        l *= keep;
#pragma unroll
                        for (int t = 0; t < CPL; ++t) o[t] *= keep;
                    }
                    const float base = m == -inf ? 0.0f : m;
                    float part = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) { p[i] = __builtin_amdgcn_exp2f(p[i] - base); part += p[i]; }
                    l += part;
                    float hi[8];
                    u32 ph[4], pl[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ph[i] = pack2<F16>(p[2 * i], p[2 * i + 1]);
                        hi[2 * i] = elem_f<F16>((bf16_t)ph[i]); hi[2 * i + 1] = elem_f<F16>((bf16_t)(ph[i] >> 16));
                        pl[i] = pack2<F16>(p[2 * i] - hi[2 * i], p[2 * i + 1] - hi[2 * i + 1]);
                    }
                    const uint4 bh = make_uint4(ph[0], ph[1], ph[2], ph[3]), bl = make_uint4(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
                    for (int t = 0; t < CPL; ++t) {
                        constexpr u32 LO = 0x05040100u, HI = 0x07060302u;
                        u32 w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(v[i >> 1][2 * (i & 1) + 1][t >> 1], v[i >> 1][2 * (i & 1)][t >> 1], t & 1 ? HI : LO);
                        if (careful < 0) {
                            const uint4 av = make_uint4(w[0], w[1], w[2], w[3]);
                            o[t] = mma32<F16>(av, bh, o[t]);
                            o[t] = mma32<F16>(av, bl, o[t]);
                        } else {
                            u32 odd[4], ps[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const u32 nf = halves_not_finite<F16>(w[i]);
                                odd[i] = w[i] & nf;
                                w[i] &= ~nf;
                                // the weight as one term that is not zero where the weight is not
                                const u32 tiny = (p[2 * i] > 0.0f && !(ph[i] & 0xffffu) ? 1u : 0u) | (p[2 * i + 1] > 0.0f && !(ph[i] >> 16) ? 0x10000u : 0u);
                                ps[i] = ph[i] | tiny;
                            }
                            const uint4 av = make_uint4(w[0], w[1], w[2], w[3]);
                            o[t] = mma32<F16>(av, bh, o[t]);
                            o[t] = mma32<F16>(av, bl, o[t]);
                            o[t] = mma32<F16>(make_uint4(odd[0], odd[1], odd[2], odd[3]), make_uint4(ps[0], ps[1], ps[2], ps[3]), o[t]);
                        }
                    }
                }
                if constexpr (!ONE) {
                    __syncthreads();                                 // (the list has been read)
                    w0 = s_next == 0x7fffffff ? -1 : s_next;
                    __syncthreads();
                }
            }
            // the waves' shares of each column meet
            __syncthreads();
            l = xor_add<32>(xor_add<16>(l));
            if (c < a.cols) {
                float* const dst = s_o + (wave * a.cols + c) * OS + 4 * g * CPL;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < CPL; t += 4) *reinterpret_cast<float4*>(dst + i * CPL + t) = make_float4(o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]);
                if (g == 0) { s_ml[(wave * a.cols + c) * 2] = m; s_ml[(wave * a.cols + c) * 2 + 1] = l; }
            }
            __syncthreads();
            bool bad = false;
            for (int it = tid; it < a.cols * (D / 8); it += 64 * W) {
                const int cc = it / (D / 8), d = it % (D / 8) * 8, r = ONE ? 0 : cc / gh, hh = ONE ? cc : cc % gh;
                if (ONE ? cc >= gh : r < ra || r >= rb) continue;
                if (careful >= 0 && r != careful) continue;
                float mm = -inf, sum = 0.0f, acc[8] = {};
                for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_ml[(w * a.cols + cc) * 2]);
                const float base = mm == -inf ? 0.0f : mm;
                for (int w = 0; w < W; ++w) {
                    const float f = __builtin_amdgcn_exp2f(s_ml[(w * a.cols + cc) * 2] - base);
                    sum = __fmaf_rn(f, s_ml[(w * a.cols + cc) * 2 + 1], sum);
#pragma unroll
                    for (int x = 0; x < 8; ++x) acc[x] = __fmaf_rn(f, s_o[(w * a.cols + cc) * OS + d + x], acc[x]);
                }
                bad |= !(fabsf(sum) < inf);
#pragma unroll
                for (int x = 0; x < 8; ++x) bad |= !(fabsf(acc[x]) < inf);
                const size_t row = (size_t)(i0 + r) * a.Hq + h * G + h0 + hh;
                if (ONE && a.splits > 1) {
                    float* const dst = a.part_o + (row * a.splits + split) * D + d;
                    *reinterpret_cast<float4*>(dst) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (row * a.splits + split) * 2) = make_float2(mm, s_seen ? sum : -1.0f);      // (-1: the row lists nothing)
                    continue;
                }
                const bool seen = (s_seen >> r & 1) != 0;            // a row that lists nothing is zero
                u32 w[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] = seen ? pack2<F16>(acc[2 * x] / sum, acc[2 * x + 1] / sum) : 0u;
                bf16_t* const dst = a.out + row * D + d;
                if (a.out_al) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                else
#pragma unroll
                    for (int x = 0; x < 8; ++x) dst[x] = (bf16_t)(w[x / 2] >> (16 * (x & 1)));
            }
            const int again = __syncthreads_or(bad);
            if (careful < 0 ? !again : careful + 1 >= rb) break;
            careful = careful < 0 ? ra : careful + 1;
        }
        ra = rb;
    }
}

// the splits of a row and head: a wave each
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_attn_merge(BlockAttnArgs a) {
    const int at = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (at >= a.n_rows * a.Hq) return;
    const int i = at / a.Hq, len = a.q_kvlen[i], req = a.q_req[i];
    if (len <= 0 || req < 0 || req >= a.n_req) return;
    const float inf = __uint_as_float(0x7f800000u);
    const float* const ml = a.part_ml + (size_t)at * a.splits * 2;
    float m = lane < a.splits ? ml[2 * lane] : -inf, s = lane < a.splits ? ml[2 * lane + 1] : 0.0f;
    const bool none = __shfl(s, 0, 64) == -1.0f;
    float top = m;
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float f = __builtin_amdgcn_exp2f(m - (top == -inf ? 0.0f : top));
    const float sum = butterfly<64>(lane < a.splits ? f * s : 0.0f);
    float acc[D / 64] = {};
    for (int z = 0; z < a.splits; ++z) {
        const float fz = __shfl(f, z, 64);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) acc[x] = __fmaf_rn(fz, a.part_o[((size_t)at * a.splits + z) * D + lane + 64 * x], acc[x]);
    }
#pragma unroll
    for (int x = 0; x < D / 64; ++x) a.out[(size_t)at * D + lane + 64 * x] = none ? 0 : f_elem<F16>(acc[x] / sum);
}

// ================================================================================================
// entry points
// ================================================================================================
#define APPEND_MANY (1 << 18)             // 16-channel pieces of a call from which on threads go through several heads
#define BY_TYPE_AND_DIM(KERN, c) \
    ((c).dtype == VOX_DTYPE_F16 ? ((c).head_dim == 128 ? (const void*)KERN<1, 128> : (const void*)KERN<1, 64>) \
                                : ((c).head_dim == 128 ? (const void*)KERN<0, 128> : (const void*)KERN<0, 64>))

static int launch_bounds(hipStream_t st, const vox_block_cache& c, const int* page, const int* slot, int n_rows) {
    if (n_rows == 0) return VOX_OK;
    BoundsArgs b{(const bf16_t*)c.kv, c.bounds, c.steps, page, slot, n_rows, c.n_pages, c.page_size, c.block, c.kv_heads};
    return launch(BY_TYPE_AND_DIM(k_block_bounds, c), dim3((n_rows + 63) / 64, c.kv_heads), 256, 0, st, b);
}

extern "C" {

int vox_block_bounds(vox_ctx* ctx, void* stream, const vox_block_cache* c, const int32_t* page, const int32_t* slot, int n_rows) {
    (void)ctx;
    if (!c) return vox_fail(VOX_ERR_INVALID, "block_bounds: no cache");
    VOX_TRY(check_cache("block_bounds", *c, true));
    VOX_TRY(check_bounds("block_bounds", *c));
    if (n_rows < 0 || (n_rows && (!page || !slot))) return vox_fail(VOX_ERR_INVALID, "block_bounds: %d rows, or no page or slot", n_rows);
    return launch_bounds((hipStream_t)stream, *c, page, slot, n_rows);
}

int vox_rope_append(vox_ctx* ctx, void* stream, const vox_rope_append_args* a) {
    (void)ctx;
    if (!a) return vox_fail(VOX_ERR_INVALID, "rope_append: no arguments");
    const vox_block_cache& c = a->cache;
    VOX_TRY(check_cache("rope_append", c, c.bounds != nullptr));
    if (c.bounds) VOX_TRY(check_bounds("rope_append", c));
    const int D = c.head_dim;
    if (D < 2 || D % 2 || D > 512) return vox_fail(VOX_ERR_INVALID, "rope_append: head_dim %d (even, 2 to 512)", D);
    if (a->n_rows < 0 || a->n_own < 0 || a->heads <= 0) return vox_fail(VOX_ERR_INVALID, "rope_append: %d rows of %d requests, %d heads", a->n_rows, a->n_own, a->heads);
    if (a->rot < 0 || a->rot % 2 || a->rot > D) return vox_fail(VOX_ERR_INVALID, "rope_append: %d of %d channels turn", a->rot, D);
    if (a->n_rows == 0) return VOX_OK;
    if (!a->q || !a->k || !a->v || !a->q_out || !a->page || !a->slot) return vox_fail(VOX_ERR_INVALID, "rope_append: an operand is NULL");
    if (a->rot && (!a->pos || !a->table || a->table_max_pos <= 0)) return vox_fail(VOX_ERR_INVALID, "rope_append: no positions or no table");
    if (((size_t)a->q | (size_t)a->k | (size_t)a->v | (size_t)a->q_out) & 1 || (a->rot && (size_t)a->table & 3)) return vox_fail(VOX_ERR_INVALID, "rope_append: an operand does not lie on its type");
    if (a->q_stride < 0 || a->k_stride < 0 || a->v_stride < 0) return vox_fail(VOX_ERR_INVALID, "rope_append: a stride is negative");
    const int heads = a->heads + 2 * c.kv_heads;
    RopeAppendArgs r{(const bf16_t*)a->q, (const bf16_t*)a->k, (const bf16_t*)a->v, (bf16_t*)a->q_out, (bf16_t*)c.kv, a->pos, a->page, a->slot, a->table, c.bounds, c.steps,
                     (long)a->q_stride, (long)a->k_stride, (long)a->v_stride, a->n_rows, a->heads, c.kv_heads, D, a->rot, a->interleave, a->table_max_pos, c.page_size, c.n_pages, c.block, heads, 0};
    const bool f16 = c.dtype == VOX_DTYPE_F16;
    // 16 channels a thread: everything on 16 bytes, and no pair of eight across the border of what turns
    const bool vec = D % 16 == 0 && a->rot % 16 == 0 && (((size_t)a->q | (size_t)a->k | (size_t)a->v | (size_t)a->q_out | (a->rot ? (size_t)a->table : 0)) & 15) == 0 &&
                     a->q_stride % 8 == 0 && a->k_stride % 8 == 0 && a->v_stride % 8 == 0;
    const bool with = vec && c.bounds && a->n_own == a->n_rows;      // the bounds in the same launch
    int64_t blocks;
    if (vec) {
        if ((int64_t)a->n_rows * heads * (D / 16) >= APPEND_MANY && heads > 8) r.slots = 8;
        blocks = ((int64_t)a->n_rows * r.slots * (D / 16) + 255) / 256;
    } else blocks = ((int64_t)a->n_rows * heads * (D / 2) + 255) / 256;
    const int64_t more = with ? ((int64_t)a->n_rows * c.kv_heads + 3) / 4 : 0;
    if (blocks + more > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "rope_append: %d rows of %d heads are more than a launch holds", a->n_rows, a->heads);
    r.append_blocks = (int)blocks;
    const void* kern;
    if (!vec) kern = f16 ? (const void*)k_rope_append_any<1> : (const void*)k_rope_append_any<0>;
#define APPEND_OF(IL) \
    (!with ? (f16 ? (const void*)k_rope_append<1, IL, 0> : (const void*)k_rope_append<0, IL, 0>) \
     : D == 128 ? (f16 ? (const void*)k_rope_append<1, IL, 128> : (const void*)k_rope_append<0, IL, 128>) \
                : (f16 ? (const void*)k_rope_append<1, IL, 64> : (const void*)k_rope_append<0, IL, 64>))
    else kern = a->interleave ? APPEND_OF(1) : APPEND_OF(0);
#undef APPEND_OF
    VOX_TRY(launch(kern, dim3((unsigned)(blocks + more)), 256, 0, (hipStream_t)stream, r));
    return c.bounds && !with ? launch_bounds((hipStream_t)stream, c, a->page, a->slot, a->n_rows) : VOX_OK;
}

static int check_select(const vox_block_select_args* a) {
    if (!a) return vox_fail(VOX_ERR_INVALID, "block_select: no arguments");
    const vox_block_cache& c = a->cache;
    if (c.n_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return vox_fail(VOX_ERR_INVALID, "block_select: %d pages of %d tokens, %d kv heads", c.n_pages, c.page_size, c.kv_heads);
    vox_block_cache k = c;
    k.kv = c.bounds;                                                // the keys are not read: the bounds stand for them
    VOX_TRY(check_cache("block_select", k, true));
    VOX_TRY(check_bounds("block_select", c));
    VOX_TRY(check_rows("block_select", c, a->rows));
    if (a->first < 0 || a->last < 1 || a->top > VOX_BLOCK_TOP_MAX || (int64_t)a->first + a->last > a->top) return vox_fail(VOX_ERR_INVALID, "block_select: top %d (up to %d), first %d, last %d (1 at least)", a->top, VOX_BLOCK_TOP_MAX, a->first, a->last);
    if ((a->rows.max_kvlen + (int64_t)c.block - 1) / c.block > VOX_BLOCK_SELECT_MAX) return vox_fail(VOX_ERR_INVALID, "block_select: %d tokens are more than %d blocks of %d", a->rows.max_kvlen, VOX_BLOCK_SELECT_MAX, c.block);
    if (a->q_stride < 0) return vox_fail(VOX_ERR_INVALID, "block_select: a stride is negative");
    return VOX_OK;
}
int64_t vox_block_select_workspace_bytes(const vox_block_select_args* a) {
    if (check_select(a) != VOX_OK) return -1;
    return 0;
}
int vox_block_select(vox_ctx* ctx, void* stream, const vox_block_select_args* a) {
    (void)ctx;
    VOX_TRY(check_select(a));
    const vox_block_cache& c = a->cache;
    const vox_block_rows& r = a->rows;
    if (r.n_rows == 0) return VOX_OK;
    if (!a->q || !a->blocks || (size_t)a->q & 1) return vox_fail(VOX_ERR_INVALID, "block_select: an operand is NULL, or does not lie on its type");
    const int most = (r.max_kvlen + c.block - 1) / c.block;
    // rows a tile: 16 while their keys take half a CU's LDS, 8 while they take most of it (4096 blocks), else (and for rows of different requests) one
    const bool many = r.n_own > 0 && r.n_rows >= 2 * r.n_own;
    const int qt = many && most <= 1024 ? 16 : many && most <= 4096 ? 8 : 1;
    const int W = qt > 1 ? 8 : most <= 512 ? 4 : 16;
    SelectArgs s{(const bf16_t*)a->q, c.bounds, c.steps, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (long)a->q_stride,
                 r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages, c.page_size, c.block, a->top, a->first, a->last, most + (qt > 1 ? SEL_PAD : 0)};
    const int64_t grid = (int64_t)((r.n_rows + qt - 1) / qt) * c.kv_heads;
    if (grid > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "block_select: %d rows of %d kv heads are more than a launch holds", r.n_rows, c.kv_heads);
#define SELECT_OF(QT, W) (c.dtype == VOX_DTYPE_F16 ? (c.head_dim == 128 ? (const void*)k_block_select<1, 128, QT, W> : (const void*)k_block_select<1, 64, QT, W>) \
                                                  : (c.head_dim == 128 ? (const void*)k_block_select<0, 128, QT, W> : (const void*)k_block_select<0, 64, QT, W>))
    const void* kern = qt == 16 ? SELECT_OF(16, 8) : qt == 8 ? SELECT_OF(8, 8) : W == 4 ? SELECT_OF(1, 4) : SELECT_OF(1, 16);
#undef SELECT_OF
    return launch(kern, dim3((unsigned)grid), 64 * W, (size_t)qt * s.stride * 4, (hipStream_t)stream, s);
}

static int check_attention(const vox_block_attention_args* a) {
    if (!a) return vox_fail(VOX_ERR_INVALID, "block_attention: no arguments");
    VOX_TRY(check_cache("block_attention", a->cache, true));
    VOX_TRY(check_rows("block_attention", a->cache, a->rows));
    if (a->top < 0 || a->top > VOX_BLOCK_TOP_MAX) return vox_fail(VOX_ERR_INVALID, "block_attention: lists of %d blocks (up to %d)", a->top, VOX_BLOCK_TOP_MAX);
    if (a->q_stride < 0) return vox_fail(VOX_ERR_INVALID, "block_attention: a stride is negative");
    return VOX_OK;
}
// How a call's rows are laid out: rows a tile, and the parts that a row's list is split into.
struct AttnShape { int per_tile, splits, head_tiles; };
static AttnShape attn_shape(const vox_block_attention_args* a, int cus) {
    const vox_block_rows& r = a->rows;
    const int G = r.heads / a->cache.kv_heads;
    AttnShape s{1, 1, (G + 15) / 16};
    if (r.n_own > 0 && r.n_rows >= 2 * r.n_own && G <= 8) { s.per_tile = 16 / G; return s; }
    const long tokens = (long)a->top * a->cache.block, blocks = (long)r.n_rows * a->cache.kv_heads * s.head_tiles;
    if (tokens > 1024) {
        long z = (2L * cus + blocks - 1) / blocks;
        const long most = (tokens + 255) / 256;
        if (z > most) z = most;
        s.splits = (int)(z < 1 ? 1 : z > 64 ? 64 : z);
    }
    return s;
}
int64_t vox_block_attention_workspace_bytes(const vox_block_attention_args* a) {
    if (check_attention(a) != VOX_OK) return -1;
    const AttnShape s = attn_shape(a, ATTN_CUS);
    return s.splits > 1 ? (int64_t)a->rows.n_rows * a->rows.heads * s.splits * (a->cache.head_dim + 2) * 4 : 0;
}
int vox_block_attention(vox_ctx* ctx, void* stream, const vox_block_attention_args* a) {
    (void)ctx;
    VOX_TRY(check_attention(a));
    const vox_block_cache& c = a->cache;
    const vox_block_rows& r = a->rows;
    if (r.n_rows == 0) return VOX_OK;
    if (!a->q || (!a->blocks && a->top) || !a->out || ((size_t)a->q | (size_t)a->out) & 1) return vox_fail(VOX_ERR_INVALID, "block_attention: an operand is NULL, or does not lie on its type");
    const AttnShape z = attn_shape(a, ATTN_CUS);
    const size_t rows = (size_t)r.n_rows * r.heads * z.splits;
    if (z.splits > 1 && (!a->workspace || (size_t)a->workspace & 15 || a->workspace_bytes < (int64_t)(rows * (c.head_dim + 2) * 4)))
        return vox_fail(VOX_ERR_INVALID, "block_attention: a workspace of %lld bytes on 16, %lld are wanted", (long long)(a->workspace ? a->workspace_bytes : 0), (long long)(rows * (c.head_dim + 2) * 4));
    const int64_t grid = (int64_t)((r.n_rows + z.per_tile - 1) / z.per_tile) * z.splits * z.head_tiles * c.kv_heads;
    if (grid > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "block_attention: %d rows of %d heads are more than a launch holds", r.n_rows, r.heads);
    const bool one = z.per_tile == 1;
    const int W = one ? 8 : 4, G = r.heads / c.kv_heads, cols = one && G < 16 ? G : 16;
    BlockAttnArgs s{(const bf16_t*)a->q, (const bf16_t*)c.kv, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (bf16_t*)a->out, (float*)a->workspace,
                    (float*)a->workspace + rows * c.head_dim, (long)a->q_stride, a->scale * 1.44269504088896340736f, r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages,
                    c.page_size, c.block, a->top, z.per_tile, z.splits, z.head_tiles, cols, ((size_t)a->q & 15) == 0 && a->q_stride % 8 == 0, ((size_t)a->out & 15) == 0};
    const size_t merge = (size_t)W * cols * (c.head_dim + 4 + 2) * 4;
    const size_t entries = (size_t)a->top * z.per_tile, lists = one ? entries * 8 : ATTN_WINDOW * 2 + (entries < ATTN_WINDOW ? entries : ATTN_WINDOW) * 8;
    const size_t lds = merge > lists ? merge : lists;
    const void* kern = one ? (c.dtype == VOX_DTYPE_F16 ? (c.head_dim == 128 ? (const void*)k_block_attn<1, 128, 8, true> : (const void*)k_block_attn<1, 64, 8, true>)
                                                       : (c.head_dim == 128 ? (const void*)k_block_attn<0, 128, 8, true> : (const void*)k_block_attn<0, 64, 8, true>))
                           : (c.dtype == VOX_DTYPE_F16 ? (c.head_dim == 128 ? (const void*)k_block_attn<1, 128, 4, false> : (const void*)k_block_attn<1, 64, 4, false>)
                                                       : (c.head_dim == 128 ? (const void*)k_block_attn<0, 128, 4, false> : (const void*)k_block_attn<0, 64, 4, false>));
    VOX_TRY(launch(kern, dim3((unsigned)grid), 64 * W, lds, (hipStream_t)stream, s));
    if (z.splits == 1) return VOX_OK;
    return launch(BY_TYPE_AND_DIM(k_block_attn_merge, c), dim3((unsigned)(((int64_t)r.n_rows * r.heads + 3) / 4)), 256, 0, (hipStream_t)stream, s);
}

}  // extern "C"
