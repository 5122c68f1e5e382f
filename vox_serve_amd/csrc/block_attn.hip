// Long contexts: rows rotated into a paged cache, the bounds of its blocks, the blocks that a row reads, and attention over them
// (voxhip.h: vox_rope_append, vox_block_bounds, vox_block_select, vox_block_attention).
#include <math.h>

#include <type_traits>

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

// lane ^ 16 and lane ^ 32, and f over a whole wave, f commutative: partners by swaps and DPP moves (vox_device.h's xor_add), not by the LDS crossbar
template <int OFF>                       // 16 or 32
__device__ __forceinline__ float xor_max(float s) {
    vox_u2 r;
    if constexpr (OFF == 32) r = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    else r = __builtin_amdgcn_permlane16_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
template <class F>
__device__ __forceinline__ u32 wave_all(u32 x, F f) {
    vox_u2 r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = f(r.x, r.y);
    r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(r.x, r.y);
    x = f(x, (u32)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xF, 0xF, false));      // lane ^ 8
    int y = __builtin_amdgcn_update_dpp((int)x, (int)x, 0x104, 0xF, 0x5, false);             // lane ^ 4
    y = __builtin_amdgcn_update_dpp(y, (int)x, 0x114, 0xF, 0xA, false);
    x = f(x, (u32)y);
    x = f(x, (u32)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x4E, 0xF, 0xF, false));       // lane ^ 2
    x = f(x, (u32)__builtin_amdgcn_update_dpp((int)x, (int)x, 0xB1, 0xF, 0xF, false));       // lane ^ 1
    return __builtin_amdgcn_readfirstlane(x);
}

// Sixteen rows of 2 D bytes in LDS: 16 bytes of a row at position chunk ^ swizzle(row), so that 16 rows' same chunk lie on all banks
template <int D>
__device__ __forceinline__ u32 tile_place(int row, int chunk) {      // byte of a tile's [16][D]
    return D == 128 ? (u32)(row * 256 + ((chunk ^ row) << 4)) : (u32)(row * 128 + ((chunk ^ (row >> 1 & 7)) << 4));
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// n and the bits of m below the lane's own
__device__ __forceinline__ int lanes_below(unsigned long long m, int n) {
    return (int)__builtin_amdgcn_mbcnt_hi((u32)(m >> 32), __builtin_amdgcn_mbcnt_lo((u32)m, (u32)n));
}

// Rows ra, ra + 1, .. of a tile that belong to one request (a lane has its row's request, -1: passed over): one past the last, and the most tokens one of them sees
__device__ __forceinline__ int run_of(int my_req, int my_len, int ra, int R, int lane, int req, int& n_most) {
    const unsigned long long same = __ballot(lane < R && my_req == req) >> ra;
    const int rb = ra + (int)__builtin_ctzll(~same);                 // (R is below 64: a zero follows)
    n_most = (int)wave_all(lane >= ra && lane < rb ? (u32)my_len : 0u, [](u32 x, u32 y) { return max(x, y); });
    return rb;
}

#define ATTN_CUS 256                     // of an MI355X

static int check_cache(const char* who, const vox_block_cache& c, bool bounds) {
    if (!c.kv) return vox_fail(VOX_ERR_INVALID, "%s: no cache", who);
    if (c.n_pages <= 0 || c.page_size <= 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return vox_fail(VOX_ERR_INVALID, "%s: %d pages of %d tokens, %d kv heads", who, c.n_pages, c.page_size, c.kv_heads);
    if (c.dtype != VOX_DTYPE_BF16 && c.dtype != VOX_DTYPE_F16) return vox_fail(VOX_ERR_INVALID, "%s: dtype %d", who, c.dtype);
    if ((size_t)c.kv & 15) return vox_fail(VOX_ERR_INVALID, "%s: the cache does not lie on 16 bytes", who);
    if (!bounds) return VOX_OK;
    if ((int64_t)c.n_pages * (c.page_size / (c.block > 0 ? c.block : 1)) * c.kv_heads > 0xffffffffll) return vox_fail(VOX_ERR_INVALID, "%s: %d pages of %d tokens and %d kv heads are 2^32 blocks or more", who, c.n_pages, c.page_size, c.kv_heads);
    if ((int64_t)c.n_pages * c.page_size > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "%s: %d pages of %d tokens are 2^31 or more", who, c.n_pages, c.page_size);
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

// The bounds of one block, by one wave: D / 8 lanes hold a key, 512 / D keys at once, eight such loads in flight.  The first `count` keys are in the cache, one more may
// come from own(l), channels 8 l .. 8 l + 7.  (A key twice changes no bound: places behind the last take the last.)
template <int F16, int D, class O>
__device__ __forceinline__ void block_bounds(int lane, const bf16_t* keys, size_t row_el, int count, bool more, int8_t* bounds, float* step_out, O own) {
    constexpr int LPT = D / 8, TPI = 64 / LPT;
    const float inf = __uint_as_float(0x7f800000u);
    const int l = lane % LPT;
    float hi[8], lo[8], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) { hi[i] = -inf; lo[i] = inf; }
    auto take = [&](const uint4& v) {
        const u32 w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = elem_f<F16>((bf16_t)(w[i / 2] >> (16 * (i % 2))));
            hi[i] = x > hi[i] ? x : hi[i];                          // (false for NaN)
            lo[i] = x < lo[i] ? x : lo[i];
            amax = fmaxf(amax, finite_abs(x));                      // (of all keys: infinities would stand in front of it in the bounds)
        }
    };
    const bf16_t* const from = keys + 8 * l;
    for (int t0 = 0; t0 < count; t0 += 8 * TPI) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = *reinterpret_cast<const uint4*>(from + (size_t)min(t0 + u * TPI + lane / LPT, count - 1) * row_el);
#pragma unroll
        for (int u = 0; u < 8; ++u) take(v[u]);
    }
    if (more) take(own(l));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (LPT == 8) { hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], 8, 64)); lo[i] = fminf(lo[i], __shfl_xor(lo[i], 8, 64)); }
        hi[i] = xor_max<32>(xor_max<16>(hi[i]));
        lo[i] = -xor_max<32>(xor_max<16>(-lo[i]));
    }
    amax = __uint_as_float(wave_all(__float_as_uint(amax), [](u32 x, u32 y) { return max(x, y); }));
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
// Bound by memory: 16384 rows of 32 + 2 x 8 heads of 128 are 411 MB with their angles, 75 us (5.5 TB/s: requests share angles), their bounds 14 us more;
// 48 rows 7 us, one row 2.3, the launch.
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
        block_bounds<F16, D>(threadIdx.x & 63, base, (size_t)a.Hkv * D, a.block - 1, true, a.bounds + to * 2 * D, a.steps + to, [&](int l) {
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
// 64 rows and a kv head a block of threads; its waves share the rows that complete a block (blocks of 16: one each).  16384 rows' 256 blocks of 64 and 8 kv heads, 34 MB: 14 us, some 7 of
// them at the memory's rate; a wave has its block's keys in flight 32 at a time.
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_bounds(BoundsArgs a) {
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), h = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int pg = -1, slot = 0;
    const bool done = n < a.n_rows && row_place(a.page, a.slot, n, a.n_pages, a.page_size, pg, slot) && (slot + 1) % a.block == 0;
    unsigned long long left = __ballot(done);
    for (int i = 0; left; ++i, left &= left - 1) {
        if ((i & 3) != wave) continue;
        const int from = __builtin_ctzll(left), p = __builtin_amdgcn_readlane(pg, from), s = __builtin_amdgcn_readlane(slot, from);
        const bf16_t* const k = a.kv + ((size_t)p * 2 * a.page_size + s + 1 - a.block) * a.Hkv * D + (size_t)h * D;
        const size_t to = ((size_t)p * a.Hkv + h) * (a.page_size / a.block) + s / a.block;
        block_bounds<F16, D>(lane, k, (size_t)a.Hkv * D, a.block, false, a.bounds + to * 2 * D, a.steps + to, [](int) { return make_uint4(0, 0, 0, 0); });
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
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top, first, last, stride, q_al, splits, stage_at;      // stage_at: byte of the waves' blocks in LDS
    u32* keys;                           // splits > 1: [row][kv head][stride]
    u32 per_magic;                       // j / per = umulhi(j, per_magic) for j < 2^16 (0: per is 1)
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
// The keys of all candidates lie in LDS: [row][stride].
// 4096 rows of a request, 16 heads on 8 of 128, 512 blocks each: 63 us, floor 7 (the product, far from what bounds it).  With
// one part left out at a time: choosing 27 us, products and the 268 MB of bounds on their way 13, q to matrix rows 8 (16 with eight lanes to a bank and one
// address for a row's maximum), the rest 18: a chain of row, pages, steps and bounds, with two blocks of threads a CU to hide it.
// One row of 2048 blocks of 2 kv heads: 5.7 us for its scores over 16 blocks of threads, 6.5 to choose; 32 rows of 512 blocks and 8 kv heads 12 us, floor 5.5.
#define SEL_PAD 8
// keys of one row, a wave's or W waves' (W > 1: all threads call): the need largest, older first where equal, written in order of their index
template <int KPL, int W>
__device__ __forceinline__ void choose(u32* key, int lo, int cand, int need, int first, int last, int have, int top, int* out, int lane, int wave, int (*red)[16]) {
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
    int turn = 0;
    auto total3 = [&](int (&n)[3]) {                                 // over the row's waves: three sums in turn, the next one cleared before this one's barrier
        if (lane < 3) atomicAdd(&red[turn][lane], lane == 0 ? n[0] : lane == 1 ? n[1] : n[2]);
        const int next = turn == 2 ? 0 : turn + 1;
        if (wave == 0 && lane < 3) red[next][lane] = 0;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 3; ++x) n[x] = __builtin_amdgcn_readfirstlane(red[turn][x]);
        turn = next;
    };
    // the need-th largest key t lies in [a, b): at least need keys reach a, fewer reach b
    least = wave_all(least, [](u32 x, u32 y) { return min(x, y); });
    most = wave_all(most, [](u32 x, u32 y) { return max(x, y); });
    if constexpr (W > 1) {
        u32* const r = reinterpret_cast<u32*>(red[3]);
        u32* const s = reinterpret_cast<u32*>(red[4]);
        if (lane == 0) { r[wave] = least; s[wave] = most; }
        if (wave == 0 && lane < 3) red[0][lane] = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) { least = min(least, r[w]); most = max(most, s[w]); }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
    }
    u32 a = least, t = least;
    unsigned long long b = (unsigned long long)most + 1;
    // A wave with many keys looks at the largest of each 128th of them first: what `need` of those reach, at least `need` keys reach, and few more (of 512 keys and 29
    // some 40).  These keys move together, and the search goes on over one or two a lane: 4096 rows of 512 blocks 63 us, 75 with every round over all keys.
    if constexpr (W == 1 && KPL >= 4) {
        constexpr int R = KPL >= 8 ? 2 : 1;                          // keys a lane that the row has room for, beside their indexes
        if (need > 0 && need <= 48 * R) {
            u32 m[2] = {k[0], k[1]};
#pragma unroll
            for (int i = 2; i < KPL; ++i) m[i & 1] = max(m[i & 1], k[i]);
            unsigned long long hi = b;
            for (int n = 128; n > need + 8 && hi - a > 1;) {
                const u32 mid = a + (u32)((hi - a) >> 1);
                const int reach = (int)__popcll(__ballot(m[0] >= mid)) + (int)__popcll(__ballot(m[1] >= mid));
                if (reach >= need) { a = mid; n = reach; } else hi = mid;
            }
            // (a = 0: lanes outside reach it)
            u32* const row = key + lo;                               // (the keys are in registers: their row is free)
            int total = 0;
            if (a > 0)
#pragma unroll
                for (int i = 0; i < KPL; ++i) {
                    const unsigned long long r = __ballot(k[i] >= a);
                    const int to = lanes_below(r, total);
                    if (k[i] >= a && to < 64 * R) { row[to] = k[i]; row[64 * R + to] = (u32)(lo + i * 64 + lane); }
                    total += (int)__popcll(r);
                }
            asm volatile("" ::: "memory");                           // (a wave's LDS instructions are in order)
            auto rest = [&](auto regs) {
                constexpr int N = decltype(regs)::value;
                u32 x[N], index[N];
#pragma unroll
                for (int i = 0; i < N; ++i) { x[i] = 64 * i + lane < total ? row[64 * i + lane] : 0; index[i] = row[64 * R + 64 * i + lane]; }
                bool exact = total == need;
                while (!exact && b - a > 1) {
                    const u32 mid = a + (u32)((b - a) >> 1);
                    int n = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) n += (int)__popcll(__ballot(x[i] >= mid));
                    if (n >= need) a = mid; else b = mid;
                    exact = n == need;
                }
                int gt = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) gt += (int)__popcll(__ballot(exact ? x[i] >= a : x[i] > a));
                int ties = need - gt, to = first;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const bool e = x[i] == a && !exact, g = exact ? x[i] >= a : x[i] > a;
                    const unsigned long long be = __ballot(e);
                    const bool take = g || (e && lanes_below(be, 0) < ties);
                    const unsigned long long bt = __ballot(take);
                    if (take) out[lanes_below(bt, to)] = (int)index[i];
                    to += (int)__popcll(bt);
                    ties -= min(ties, (int)__popcll(be));
                }
                for (int j = lane; j < first; j += 64) out[j] = j;
                for (int j = lane; j < last; j += 64) out[top - last + j] = have - last + j;
            };
            if (total >= need && total <= 64) return rest(std::integral_constant<int, 1>{});
            if constexpr (R == 2) if (total >= need && total <= 128) return rest(std::integral_constant<int, 2>{});
            t = a;
        }
    }
    bool exact = need == 0;                                          // exactly `need` keys reach t: no ties to break
    while (!exact && b - a > 1) {
        if constexpr (W > 1) {
            // three cuts a round: a round is its barrier, not its compares
            const u32 len = (u32)((b - a) >> 2), cut[3] = {a + max(len, 1u), a + max(2 * len, 1u), a + max(3 * len, 1u)};
            int n[3] = {0, 0, 0};
#pragma unroll
            for (int i = 0; i < KPL; ++i)
#pragma unroll
                for (int x = 0; x < 3; ++x) n[x] += (int)__popcll(__ballot(k[i] >= cut[x]));
            total3(n);
            if (n[0] < need) b = cut[0];
            else if (n[1] < need) { a = cut[0]; b = cut[1]; exact = n[0] == need; }
            else if (n[2] < need) { a = cut[1]; b = cut[2]; exact = n[1] == need; }
            else { a = cut[2]; exact = n[2] == need; }
        } else {
            const u32 mid = a + (u32)((b - a) >> 1);
            int n = 0;
#pragma unroll
            for (int i = 0; i < KPL; ++i) n += (int)__popcll(__ballot(k[i] >= mid));      // (mid > least >= 0: lanes outside, 0, never reach it)
            if (n >= need) a = mid; else b = mid;
            exact = n == need;
        }
        t = a;
    }
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
    int at = first + gt_before + min(eq_before, ties);
    ties = max(ties - eq_before, 0);
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
        if (c0 + i * 64 >= cand || need == 0) break;
        const bool in = c0 + i * 64 + lane < cand, e = in && !exact && k[i] == t, g = in && (exact ? k[i] >= t : k[i] > t);
        const unsigned long long be = __ballot(e);
        const bool take = g || (e && lanes_below(be, 0) < ties);
        const unsigned long long bt = __ballot(take);
        if (take) out[lanes_below(bt, at)] = lo + c0 + i * 64 + lane;
        at += (int)__popcll(bt);
        ties -= min(ties, (int)__popcll(be));
    }
    if (W == 1 || wave == 0) {
        for (int j = lane; j < first; j += 64) out[j] = j;
        for (int j = lane; j < last; j += 64) out[top - last + j] = have - last + j;
    }
}

// QT > 1: tiles of QT rows, a wave a row in the choice; QT == 1: a row, all waves together
// SPLIT (QT == 1): the scores alone, of one part of the row's blocks, into the workspace
// NT: tiles of 16 blocks that a wave brings to its part of LDS at a time, in rows of memory (a lane's 16 bytes of a block beside the next block's 16 would go through the
// address unit at a quarter of the rate); 0, where the keys leave no room for it: straight to registers
template <int F16, int D, int QT, int W, bool SPLIT, int NT>
__global__ __launch_bounds__(64 * W, QT == 16 ? 4 : 2) void k_block_select(SelectArgs a) {
    constexpr int MT = (2 * QT + 15) / 16, KS = 2 * D / 64;          // tiles of 16 product rows, steps of 64 numbers
    extern __shared__ __attribute__((aligned(16))) u32 keys[];       // [QT][a.stride]; before: [QT][D], N and P of a channel in the halves
    __shared__ __attribute__((aligned(16))) int8_t s_a[MT * 16][2 * D];
    __shared__ int s_len[QT], s_req[QT], red[5][16];
    __shared__ u32 s_amax[QT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int h = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv, i0 = (SPLIT ? tile / a.splits : tile) * QT, R = min(QT, a.n_rows - i0), G = a.Hq / a.Hkv, per = a.page_size / a.block;
    const int split = SPLIT ? tile % a.splits : 0;
    if (tid < QT) {
        int n = 0, r = -1;
        if (tid < R) {
            n = a.q_kvlen[i0 + tid];
            r = a.q_req[i0 + tid];
            if (n <= 0 || r < 0 || r >= a.n_req || a.max_kvlen <= 0) { n = 0; r = -1; }
            n = min(n, a.max_kvlen);
        }
        s_len[tid] = n; s_req[tid] = r;
        s_amax[tid] = 0;
    }
    // The first row's pages, steps and first tile of bounds: asked for here, a link of the chain before each barrier that waits for the memory anyway.
    const int e_req = a.q_req[i0];
    const bool early = a.q_kvlen[i0] > 0 && e_req >= 0 && e_req < a.n_req && a.max_kvlen > 0;
    const int e_p0 = early ? a.indptr[e_req] : 0, e_np = early ? a.indptr[e_req + 1] - e_p0 : 0;
    auto page_of = [&](int j, int& pj, int p0, int np) {
        pj = a.per_magic ? (int)__umulhi((u32)j, a.per_magic) : j;
        const int pg = pj < np ? a.indices[p0 + pj] : -1;
        return pg;
    };
    auto block_of = [&](int j, int pj, int pg, float& step) {
        const bool ok = pg >= 0 && pg < a.n_pages;
        const u32 at = ok ? ((u32)pg * a.Hkv + h) * per + (j - pj * per) : 0;
        step = ok ? a.steps[at] : __uint_as_float(0x7fc00000u);      // (NaN: a block without a page)
        return at;
    };
    const int e_j = a.first + (split * W + wave) * 64 + lane;
    int e_pj;
    const int e_pg = page_of(e_j, e_pj, e_p0, e_np);
    for (int x = tid; x < QT * D; x += 64 * W) keys[x] = 0;
    if constexpr (QT < 8) for (int x = tid; x < (MT * 16 - 2 * QT) * 2 * D / 4; x += 64 * W) reinterpret_cast<int*>(s_a[2 * QT])[x] = 0;
    // P and N of the rows: eight channels of a head a thread
    const int chunks = G * D / 8;
    auto piece = [&](int it) {
        const bf16_t* const q = a.q + (size_t)(i0 + it / chunks) * a.q_stride + (size_t)h * G * D + it % chunks * 8;
        if (a.q_al) return *reinterpret_cast<const uint4*>(q);
        return make_uint4((u32)q[0] | ((u32)q[1] << 16), (u32)q[2] | ((u32)q[3] << 16), (u32)q[4] | ((u32)q[5] << 16), (u32)q[6] | ((u32)q[7] << 16));
    };
    const uint4 mine = tid < R * chunks ? piece(tid) : make_uint4(0, 0, 0, 0);
    __syncthreads();
    float e_step;
    const u32 e_at = block_of(e_j, e_pj, e_pg, e_step);
    for (int it = tid; it < R * chunks; it += 64 * W) {
        const uint4 x = it == tid ? mine : piece(it);
        const u32 w[4] = {x.x, x.y, x.z, x.w};
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(elem_f<F16>((bf16_t)(w[e / 2] >> (16 * (e % 2))))));
        u32 most = __float_as_uint(amax);                            // (pieces of a row come in eights: one of them writes)
        most = max(most, (u32)__builtin_amdgcn_update_dpp((int)most, (int)most, 0xB1, 0xF, 0xF, false));       // lane ^ 1
        most = max(most, (u32)__builtin_amdgcn_update_dpp((int)most, (int)most, 0x4E, 0xF, 0xF, false));       // lane ^ 2
        most = max(most, (u32)__builtin_amdgcn_update_dpp((int)most, (int)most, 0x141, 0xF, 0xF, false));      // lane ^ 7
        if (lane % 8 == 0) atomicMax(&s_amax[it / chunks], most);
    }
    __syncthreads();
    const u32 stage_at = a.stage_at + wave * NT * 32 * D, stage0 = (u32)(size_t)(__attribute__((address_space(3))) u32*)keys + stage_at, place = tile_place<D>(c, g);
    const char* const stage = reinterpret_cast<const char*>(keys) + stage_at;
    auto fetch = [&](int u0, u32 at) {                               // NT tiles of a step's four, from u0 on
        constexpr int LPR = D / 8, PIECES = 32 * D / 1024;           // lanes a row, loads a tile
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int row = i * (64 / LPR) + lane / LPR, chunk = lane % LPR ^ (D == 128 ? row : row >> 1 & 7);      // (what tile_place puts at this lane's position)
                const u32 from = (u32)__shfl((int)at, 16 * (u0 + u) + row, 64);
                lds_dma16(a.bounds + (size_t)from * (2 * D) + 16 * chunk, stage0 + (u32)(u * 32 * D + i * 1024));
            }
    };
    if constexpr (NT > 0) fetch(0, e_at);
    for (int it = tid; it < R * chunks; it += 64 * W) {
        const uint4 x = it == tid ? mine : piece(it);
        const u32 w[4] = {x.x, x.y, x.z, x.w};
        const int r = it / chunks, d = it % chunks % (D / 8) * 8;
        const float inv = 1.0f / step_of(__uint_as_float(s_amax[r]));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int s = q_steps(elem_f<F16>((bf16_t)(w[e / 2] >> (16 * (e % 2)))), inv);
            atomicAdd(&keys[r * D + (e * (D / 8) + d / 8 + 16 * r) % D], s >= 0 ? (u32)s : (u32)-s << 16);      // (neighbouring lanes and rows on banks of their own)
        }
    }
    __syncthreads();
    for (int x = tid; x < R * D; x += 64 * W) {
        const int r = x / D, d = x % D;
        const u32 both = keys[r * D + (d % 8 * (D / 8) + d / 8 + 16 * r) % D];
        const int p = (int)(both & 0xffffu), m = -(int)(both >> 16);
        s_a[2 * r][d] = (int8_t)(p & 63); s_a[2 * r + 1][d] = (int8_t)(p >> 6);
        s_a[2 * r][D + d] = (int8_t)(m & 63); s_a[2 * r + 1][D + d] = (int8_t)(m >> 6);
    }
    __syncthreads();
    i32x4 av[MT][KS];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < KS; ++s) av[t][s] = *reinterpret_cast<const i32x4*>(&s_a[16 * t + c][64 * s + 16 * g]);

    if constexpr (NT > 0) dma_wait();                                // (also where no step follows: nothing may be on its way to LDS that is let go of)
    const int my_req = lane < R ? s_req[lane] : -1, my_len = lane < R ? s_len[lane] : 0;
    for (int ra = 0; ra < R;) {
        const int req = __builtin_amdgcn_readlane(my_req, ra);
        if (req < 0) { ++ra; continue; }
        const int p0 = early && ra == 0 ? e_p0 : a.indptr[req], np = early && ra == 0 ? e_np : a.indptr[req + 1] - p0;
        int n_most;
        int rb = 1;
        if constexpr (QT == 1) n_most = __builtin_amdgcn_readfirstlane(my_len);
        else rb = run_of(my_req, my_len, ra, R, lane, req, n_most);
        const int have = (n_most - 1) / a.block + 1, j1 = have > a.top ? have - a.last : 0;      // blocks to score: [first, j1)
        // 64 blocks a step: a lane looks up one of them, four tiles of 16 go through the product
        u32* const dst0 = SPLIT ? a.keys + ((size_t)i0 * a.Hkv + h) * a.stride : keys;
        for (int j0 = a.first + (split * W + wave) * 64; j0 < j1; j0 += (SPLIT ? a.splits : 1) * W * 64) {
            u32 at = e_at;
            float step = e_step;
            const bool ready = early && ra == 0 && j0 == a.first + (split * W + wave) * 64;
            if (!ready) {
                int pj;
                const int j = j0 + lane, pg = page_of(j, pj, p0, np);
                at = block_of(j, pj, pg, step);
            }
            auto score = [&](int u, const i32x4 (&b)[KS]) {
                const float st = __shfl(step, 16 * u + c, 64);
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    i32x4 s4 = {0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < KS; ++s) s4 = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[t][s], b[s], s4, 0, 0, 0);
                    u32* const dst = dst0 + (size_t)(8 * t + 2 * g) * a.stride + j0 + 16 * u + c;      // product rows 4 g + 2 x, + 1: query row 8 t + 2 g + x
                    if (QT == 1 && g) continue;
#pragma unroll
                    for (int x = 0; x < (QT == 1 ? 1 : 2); ++x)
                        if (j0 + 16 * u + c < j1) dst[x * a.stride] = st == st ? score_key((float)(s4[2 * x] + 64 * s4[2 * x + 1]) * st) : 0;
                }
            };
            if constexpr (NT > 0) {
#pragma unroll
                for (int u0 = 0; u0 < 4; u0 += NT) {
                    if (j0 + 16 * u0 >= j1) break;
                    if (u0 || !ready) fetch(u0, at);
                    dma_wait();
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        i32x4 b[KS];
#pragma unroll
                        for (int s = 0; s < KS; ++s) b[s] = *reinterpret_cast<const i32x4*>(stage + u * 32 * D + (place ^ 64 * s));
                        score(u0 + u, b);
                    }
                }
            } else {
                i32x4 b[4][KS];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const i32x4* const src = reinterpret_cast<const i32x4*>(a.bounds + (size_t)(u32)__shfl((int)at, 16 * u + c, 64) * (2 * D)) + g;
#pragma unroll
                    for (int s = 0; s < KS; ++s) b[u][s] = src[4 * s];
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (j0 + 16 * u >= j1) break;
                    score(u, b[u]);
                }
            }
        }
        if constexpr (SPLIT) return;
        __syncthreads();
        for (int r = ra + (QT > 1 ? wave : 0); r < rb; r += QT > 1 ? W : 1) {
            const int mine = (__builtin_amdgcn_readlane(my_len, r) - 1) / a.block + 1, cand = mine - a.first - a.last, need = a.top - a.first - a.last;
            int* const out = a.blocks + ((size_t)(i0 + r) * a.Hkv + h) * a.top;
            if (mine <= a.top) {
                for (int j = QT > 1 ? lane : tid; j < a.top; j += QT > 1 ? 64 : 64 * W) out[j] = j < mine ? j : -1;
                continue;
            }
            u32* const key = keys + (size_t)r * a.stride;
            constexpr int GW = QT > 1 ? 1 : W;
#define CHOOSE(KPL) choose<KPL, GW>(key, a.first, cand, need, a.first, a.last, mine, a.top, out, lane, wave, red)
            constexpr int MOST = QT == 16 ? 16 : QT == 8 ? 64 : W == 4 ? 2 : W == 8 ? 8 : 32;      // by 64 GW: the blocks that the launch was chosen for
            if (cand <= 2 * 64 * GW) { CHOOSE(2); continue; }
            if constexpr (MOST > 2) if (cand <= 4 * 64 * GW) { CHOOSE(4); continue; }
            if constexpr (MOST > 4) if (cand <= 8 * 64 * GW) { CHOOSE(8); continue; }
            if constexpr (MOST > 8) if (cand <= 16 * 64 * GW) { CHOOSE(16); continue; }
            if constexpr (MOST > 16) if (cand <= 32 * 64 * GW) { CHOOSE(32); continue; }
            if constexpr (MOST > 32) CHOOSE(64);
#undef CHOOSE
        }
        __syncthreads();
        ra = rb;
    }
}

// a row and kv head whose keys lie in the workspace
template <int W>
__global__ __launch_bounds__(64 * W) void k_block_choose(SelectArgs a) {
    __shared__ int red[5][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = blockIdx.x / a.Hkv, req = a.q_req[i];
    int n = a.q_kvlen[i];
    if (n <= 0 || req < 0 || req >= a.n_req || a.max_kvlen <= 0) return;
    n = min(n, a.max_kvlen);
    int* const out = a.blocks + (size_t)blockIdx.x * a.top;
    u32* const key = a.keys + (size_t)blockIdx.x * a.stride;
    const int mine = (n - 1) / a.block + 1, cand = mine - a.first - a.last, need = a.top - a.first - a.last;
    if (mine <= a.top) {
        for (int j = tid; j < a.top; j += 64 * W) out[j] = j < mine ? j : -1;
        return;
    }
#define CHOOSE(KPL) choose<KPL, W>(key, a.first, cand, need, a.first, a.last, mine, a.top, out, lane, wave, red)
    if (cand <= 2 * 64 * W) CHOOSE(2);
    else if (cand <= 4 * 64 * W) CHOOSE(4);
    else if (cand <= 8 * 64 * W) CHOOSE(8);
    else CHOOSE(32);
#undef CHOOSE
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
// Maximum and sum of a column stay with its lanes (online softmax, exponents of two, fp32).  A weight enters as the sum of three bf16 terms or of two fp16 ones: all
// that fp32 has of it.  (One term would cost as much as the output's own rounding; two of bf16 drop 2^-17 of a weight, which shows where values cancel.  The third costs a chunk of
// 1024 rows of 2048 tokens 140 us for 129, a row nothing that can be measured.)
// What a column must not see is kept from it by its score alone (weight 0), which holds as long as V is finite; where a result is not, the rows are gone through
// again one by one in the same order with V's masked tokens as zero, and a value that is not finite multiplied by the weight as one term (an infinity times
// several of them would be inf - inf).  Rows that see no such value come out bit for bit as if it were not there.
// What bounds it, and measured (bf16, dim 128, unless said): 64 rows of 2048 tokens, 32 heads on 8 of 64, fp16: 50 us for 268 MB, 5.4 TB/s - the memory.  4 rows of 8192, 32 heads on 2:
// 9.7 us in 32 parts and 3.9 to join them, 34 MB - the launches and one pass of latency.  A row of 512 tokens, 16 heads on 8: 7.9 us - 262 KB for each of eight CUs, which at
// the 35 bytes a ns that one draws are 7.5.
// A chunk of 1024 rows of 2048 tokens, 16 heads on 8: 140 us, 17 GFLOP (34 with the weights' three terms): tiles of 16 rows meet all that any of them lists, some
// 3.5 times one row's list, and a tile's tokens are masked, weighed and moved by vector instructions for 32 columns only.
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
    float scale2;                        // |scale| log2 e, LEAST_SCALE2 at least (a lower score is a larger one where the scale is negative: q changes its sign)
    int n_rows, n_req, Hq, Hkv, max_kvlen, n_pages, page_size, block, top;
    int splits, head_tiles, cols, q_al, out_al, negate, k_at;      // k_at: byte of the waves' K in LDS (rows of several)      // cols: columns of a wave in the merge's LDS
};
// The smallest number above zero: a masked score, -infinity, times it is what zero would not make of it, and the largest score times it is nothing (2^-21).
#define LEAST_SCALE2 1.4012984643e-45f
#define ATTN_WINDOW 4096                 // blocks whose rows' bits lie in LDS at a time (rows of several: 8 KB)

// The entries of a row's list that count, 64 at a time, by one wave: f(j, counts) for every lane.  first: the lane's entry of the first 64.
template <class F>
__device__ __forceinline__ void row_entries(const int* list, int first, int top, int have, int lane, F f) {
    int carry = -1;
    for (int e0 = 0; e0 < top; e0 += 64) {
        const int j = e0 == 0 ? first : e0 + lane < top ? list[e0 + lane] : -1;
        int most = j;                                                // the largest entry up to this one
        const int prev = __shfl_up(j, 1, 64);
        if (__ballot(lane && j >= 0 && (j <= prev || prev < 0)))     // (not simply ascending)
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
__device__ __forceinline__ int first_entry(const int* list, int top, int lane) { return lane < top ? list[lane] : -1; }

// A tile is 16 tokens.  K comes to a wave's own part of LDS (memory to LDS, no registers, no barrier: the wave waits for its own) and from there to the product's lanes: a lane has
// 16 bytes of a token, its neighbour the next token's, and loads of that pattern go through at 16 bytes a clock and CU, a quarter of what rows in order do (the chunk of
// 1024 rows was held up by it 77 % of its time, a row's block of threads drew 35 bytes a ns).
template <int D>
struct KLane {
    static constexpr int PIECES = 32 * D / 1024;                     // wave loads a tile: 64 lanes of 16 bytes, 512 / D rows
    u32 from, step, at;                                              // the lane's byte of a tile's first piece in memory and of each piece's further rows; its place of step 0
    __device__ __forceinline__ KLane(int lane, u32 row_bytes) {
        const int r = lane / (D / 8);
        from = (u32)r * row_bytes;
        step = lane % (D / 8);
        at = tile_place<D>(lane & 15, lane >> 4);
    }
    // a tile's K on its way: base its first token's (scalar), to LDS byte `to` (scalar)
    __device__ __forceinline__ void fetch(const char* base, u32 row_bytes, u32 to, int lane) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = i * (512 / D) + lane / (D / 8);            // (what tile_place puts at this lane's position)
            const u32 chunk = D == 128 ? step ^ (u32)r : step ^ (u32)(r >> 1 & 7);
            lds_dma16(base + (size_t)(i * (512 / D)) * row_bytes, from + 16 * chunk, to + 1024 * i);
        }
    }
    // scores of a tile of columns: step s of the lane's token at `at` ^ 64 s (the step's bits and the chunk's are apart)
    template <int F16, class Q>
    __device__ __forceinline__ f32x4 scores(const char* tile, Q q) const {
        f32x4 s4 = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < D / 32; ++s) s4 = mma32<F16>(*reinterpret_cast<const uint4*>(tile + (at ^ 64 * s)), q(s), s4);
        return s4;
    }
};
// T tiles' V as a wave's registers
template <int D, int T>
struct VTiles {
    static constexpr int CPL = D / 16;
    u32 v[T][4][CPL / 2];
    // (a scalar base and 32 bits a lane)
    __device__ __forceinline__ void load(int x, const char* vb, size_t row_bytes, u32 off) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const char* const src = vb + i * row_bytes + off;
            if constexpr (CPL == 8) {
                const uint4 t = *reinterpret_cast<const uint4*>(src);
                v[x][i][0] = t.x; v[x][i][1] = t.y; v[x][i][2] = t.z; v[x][i][3] = t.w;
            } else {
                const uint2 t = *reinterpret_cast<const uint2*>(src);
                v[x][i][0] = t.x; v[x][i][1] = t.y;
            }
        }
    }
    // V of the tile's tokens from `from` on is zero (the others may hold anything: weight 0 times it would not be 0)
    __device__ __forceinline__ void drop_v(int x, int from, int g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < CPL / 2; ++w) v[x][i][w] = 4 * g + i >= from ? 0u : v[x][i][w];
    }
    // V^T's rows of the product over tiles 2 y and 2 y + 1: channel CPL c + t of the lane's eight tokens
    __device__ __forceinline__ uint4 vt(int y, int t) const {
        const u32 sel = t & 1 ? 0x07060302u : 0x05040100u;
        u32 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(v[2 * y + (i >> 1)][2 * (i & 1) + 1][t >> 1], v[2 * y + (i >> 1)][2 * (i & 1)][t >> 1], sel);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
// A tile of columns against T tiles of tokens.  sees[x]: how many of the lane's tokens 4 g, 4 g + 1, .. of tile x its column sees (any number: 4 and more are all).
// m: the exponent's base, in powers of two.  It need not be the maximum, only near enough that no weight passes 2^8: a lane looks at its own scores alone, and the
// columns' lanes meet only when one of them is that far above (the first time, and a few times more); a column without such a lane keeps its base and its sums.  A tile is masked as a whole, by the base, unless the
// column's last token lies in it.  What was a third more vector instructions a tile is the same to fp32 rounding.  CAREFUL: every score is masked, and
// V that is not finite meets the weight as one term.
#define ATTN_AHEAD 8.0f
#define ATTN_LIFT 7.0f                   // fp16: weights 2^7 up, 2^15 at most, so that small ones keep their bits (2^17 tokens of a weight below 2^-24 would else be lost together)
__device__ __forceinline__ float vmax(float x, float y) {            // (fmaxf of values that are no signalling NaN: without the two instructions that would quiet them)
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
    return r;
}
// A weight as a sum of 16-bit terms that has its 24 bits: three of bf16, or two of fp16, whose sum is off by 2^-23 of it at most (the half step of what is no more than a half step)
template <int F16>
struct Terms {
    static constexpr int N = F16 ? 2 : 3;
    uint4 w[N];
};
// the weights of T tiles of scores in terms (one: the first, not zero where the weight is not); o and l go to a new base if they have to
template <int F16, int D, int T, bool CAREFUL>
__device__ __forceinline__ void weigh(f32x4 (&s4)[T], const int (&sees)[T], float scale2, float& m, float& l, f32x4 (&o)[D / 16], Terms<F16> (&b)[T / 2], uint4 (&one)[T / 2]) {
    const float inf = __uint_as_float(0x7f800000u);
    bool part = CAREFUL;
#pragma unroll
    for (int x = 0; x < T; ++x) part |= sees[x] > 0 && sees[x] < 4;
    if (__ballot(part)) {
#pragma unroll
        for (int x = 0; x < T; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) s4[x][i] = i < sees[x] ? s4[x][i] : -inf;
    }
    float top = -inf;
#pragma unroll
    for (int x = 0; x < T; ++x) top = vmax(top, sees[x] > 0 ? vmax(vmax(s4[x][0], s4[x][1]), vmax(s4[x][2], s4[x][3])) : -inf);
    top *= scale2;
    if (__ballot(top > m + ATTN_AHEAD)) {
        // (only the columns that ask for it: a column's base, and with it the rounding of its weights, goes by its own scores alone)
        const float most = xor_max<32>(xor_max<16>(top)), now = most > m + ATTN_AHEAD ? most : m, keep = __builtin_amdgcn_exp2f(m - (now == -inf ? 0.0f : now));
        m = now;
        l *= keep;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[t] *= keep;
    }
    const float base = m == -inf ? 0.0f : (F16 ? ATTN_LIFT : 0.0f) - m;
    float p[4 * T], sum[T];
#pragma unroll
    for (int x = 0; x < T; ++x) {
        const float b = sees[x] > 0 ? base : -inf;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[4 * x + i] = __builtin_amdgcn_exp2f(__fmaf_rn(s4[x][i], scale2, b));
        sum[x] = (p[4 * x] + p[4 * x + 1]) + (p[4 * x + 2] + p[4 * x + 3]);
    }
#pragma unroll
    for (int x = 0; x < T; ++x) l += sum[x];
#pragma unroll
    for (int y = 0; y < T / 2; ++y) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = p[8 * y + i];
#pragma unroll
        for (int n = 0; n < Terms<F16>::N; ++n) {
            u32 t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                t[i] = pack2<F16>(w[2 * i], w[2 * i + 1]);
                if (n + 1 < Terms<F16>::N) {                         // (what a term leaves is exact)
                    w[2 * i] -= elem_f<F16>((bf16_t)t[i]);
                    w[2 * i + 1] -= elem_f<F16>((bf16_t)(t[i] >> 16));
                }
            }
            b[y].w[n] = make_uint4(t[0], t[1], t[2], t[3]);
            if constexpr (CAREFUL) if (n == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) t[i] |= (p[8 * y + 2 * i] > 0.0f && !(t[i] & 0xffffu) ? 1u : 0u) | (p[8 * y + 2 * i + 1] > 0.0f && !(t[i] >> 16) ? 0x10000u : 0u);
                one[y] = make_uint4(t[0], t[1], t[2], t[3]);
            }
        }
    }
}
// o += V^T P^T over a pair of tiles; vt(t): channel CPL c + t of the lane's eight tokens
template <int F16, int D, bool CAREFUL, class V>
__device__ __forceinline__ void weighted(V vt, const Terms<F16>& b, const uint4& one, f32x4 (&o)[D / 16]) {
    if constexpr (CAREFUL) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            const uint4 a = vt(t), odd = make_uint4(a.x & halves_not_finite<F16>(a.x), a.y & halves_not_finite<F16>(a.y), a.z & halves_not_finite<F16>(a.z), a.w & halves_not_finite<F16>(a.w));
            const uint4 fine = make_uint4(a.x ^ odd.x, a.y ^ odd.y, a.z ^ odd.z, a.w ^ odd.w);
            o[t] = mma32<F16>(odd, one, o[t]);
#pragma unroll
            for (int n = 0; n < Terms<F16>::N; ++n) o[t] = mma32<F16>(fine, b.w[n], o[t]);
        }
    } else {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            const uint4 a = vt(t);
#pragma unroll
            for (int n = 0; n < Terms<F16>::N; ++n) o[t] = mma32<F16>(a, b.w[n], o[t]);
        }
    }
}
// a tile of columns of one wave, into the merge's LDS: s_o [wave][column][D + 4], s_ml [wave][column]
template <int D>
__device__ __forceinline__ void put_columns(float* s_o, float2* s_ml, int wave, int cols, int c, int g, float m, float l, const f32x4 (&o)[D / 16]) {
    constexpr int CPL = D / 16;
    l = xor_add<32>(xor_add<16>(l));
    if (c >= cols) return;
    float* const dst = s_o + (wave * cols + c) * (D + 4) + 4 * g * CPL;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < CPL; t += 4) *reinterpret_cast<float4*>(dst + i * CPL + t) = make_float4(o[t][i], o[t + 1][i], o[t + 2][i], o[t + 3][i]);
    if (g == 0) s_ml[wave * cols + c] = make_float2(m, l);
}
// four channels of a column of all waves; false: not finite
template <int D, int W>
__device__ __forceinline__ bool merge_columns(const float* s_o, const float2* s_ml, int cols, int cc, int d, float& m, float& sum, float (&acc)[4]) {
    const float inf = __uint_as_float(0x7f800000u);
    float2 ml[W];
    float4 o[W];
#pragma unroll
    for (int w = 0; w < W; ++w) { ml[w] = s_ml[w * cols + cc]; o[w] = *reinterpret_cast<const float4*>(s_o + (w * cols + cc) * (D + 4) + d); }
    m = -inf; sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, ml[w].x);
    const float base = m == -inf ? 0.0f : m;
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml[w].x - base);
        sum = __fmaf_rn(f, ml[w].y, sum);
        acc[0] = __fmaf_rn(f, o[w].x, acc[0]); acc[1] = __fmaf_rn(f, o[w].y, acc[1]); acc[2] = __fmaf_rn(f, o[w].z, acc[2]); acc[3] = __fmaf_rn(f, o[w].w, acc[3]);
    }
    return fabsf(sum) < inf && fabsf(acc[0]) < inf && fabsf(acc[1]) < inf && fabsf(acc[2]) < inf && fabsf(acc[3]) < inf;
}
// acc / sum (by one reciprocal: 2^-23 more beside the output's half step, 2^-8 or 2^-11), or zero where a row lists nothing
template <int F16>
__device__ __forceinline__ void store_columns(bf16_t* dst, int aligned, bool seen, float sum, const float (&acc)[4]) {
    const float r = 1.0f / sum;
    u32 w[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) w[x] = seen ? pack2<F16>(acc[2 * x] * r, acc[2 * x + 1] * r) : 0u;
    if (aligned) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else
#pragma unroll
        for (int x = 0; x < 4; ++x) dst[x] = (bf16_t)(w[x / 2] >> (16 * (x & 1)));
}
// the lane's part of a column's q
template <int D>
__device__ __forceinline__ void load_q(uint4 (&q)[D / 32], const bf16_t* src, int aligned, bool col, int negate) {
    if (aligned) {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) q[s] = *reinterpret_cast<const uint4*>(src + 32 * s);
    } else {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            u32 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (u32)src[32 * s + 2 * i] | ((u32)src[32 * s + 2 * i + 1] << 16);
            q[s] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
#pragma unroll
    for (int s = 0; s < D / 32; ++s) q[s] = col ? q[s] : make_uint4(0, 0, 0, 0);
    if (negate) {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) q[s] = make_uint4(q[s].x ^ 0x80008000u, q[s].y ^ 0x80008000u, q[s].z ^ 0x80008000u, q[s].w ^ 0x80008000u);
    }
}

// A row (and up to 16 of its heads of a kv head); its list split over `splits` blocks of threads.  A wave takes 64 tokens at a time, all of their K and V asked for at
// once, K first.  A list of up to 64 entries lies in each wave's lanes (LONG: in LDS).
template <int F16, int D, int W, bool LONG>
__global__ __launch_bounds__(64 * W, 1) void k_block_attn_row(BlockAttnArgs a) {
    constexpr int CPL = D / 16, T = 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const float inf = __uint_as_float(0x7f800000u);
    // block -> (kv head, tile of heads, split, row): neighbours are kv heads, so that a die's L2 keeps its heads' tokens
    int id = blockIdx.x;
    const int h = id % a.Hkv; id /= a.Hkv;
    const int ht = id % a.head_tiles; id /= a.head_tiles;
    const int split = id % a.splits, i = id / a.splits;
    const int* const from = a.blocks + ((size_t)i * a.Hkv + h) * a.top;
    const int first = first_entry(from, a.top, lane);
    int n = a.q_kvlen[i];
    const int req = a.q_req[i], G = a.Hq / a.Hkv, h0 = ht * 16, gh = min(G - h0, 16);
    uint4 q[D / 32];
    load_q<D>(q, a.q + (size_t)i * a.q_stride + (size_t)(h * G + h0 + (c < gh ? c : 0)) * D + 8 * g, a.q_al, c < gh, a.negate);
    if (n <= 0 || req < 0 || req >= a.n_req || a.max_kvlen <= 0) return;
    n = min(n, a.max_kvlen);
    const int p0 = a.indptr[req], np = a.indptr[req + 1] - p0, per = a.page_size / a.block, have = (n - 1) / a.block + 1;
    const int sub_shift = a.block == 16 ? 0 : a.block == 32 ? 1 : a.block == 64 ? 2 : 3;
    const size_t row_el = (size_t)a.Hkv * D, v_el = (size_t)a.page_size * row_el;
    const bf16_t* const kv = a.kv + (size_t)h * D;
    // the entries that count: their block, and its first token's place
    uint2* const list = reinterpret_cast<uint2*>(lds);
    int count = 0;
    u32 e_block = 0, e_at = 0;
    auto entry = [&](int j, bool ok, u32& at) {
        const int pj = j / per;
        int pg = -1;
        if (ok && pj < np) pg = a.indices[p0 + pj];
        at = (u32)pg * 2 * a.page_size + (u32)(j - pj * per) * a.block;
        return pg >= 0 && pg < a.n_pages;
    };
    if constexpr (LONG) {
        if (wave == 0) {
            row_entries(from, first, a.top, have, lane, [&](int j, bool ok) {
                u32 at;
                ok = entry(j, ok, at);
                const unsigned long long b = __ballot(ok);
                if (ok) list[count + __popcll(b & ((1ull << lane) - 1))] = make_uint2((u32)j, at);
                count += __popcll(b);
            });
            if (lane == 0) s_count = count;
        }
        __syncthreads();
        count = __builtin_amdgcn_readfirstlane(s_count);
    } else {
        row_entries(from, first, a.top, have, lane, [&](int j, bool ok) {
            ok = entry(j, ok, e_at);
            e_block = (u32)j;
            const unsigned long long b = __ballot(ok);
            count = (int)__popcll(b);
            if (b & (b + 1)) {                                       // (not all in front: they move there)
                const int rank = (int)__popcll(b & ((1ull << lane) - 1)), to = 4 * (ok ? rank : 63 - (lane - rank));
                e_block = __builtin_amdgcn_ds_permute(to, e_block);
                e_at = __builtin_amdgcn_ds_permute(to, e_at);
            }
        });
        count = __builtin_amdgcn_readfirstlane(count);
    }
    const u32 list_bytes = LONG ? (u32)(a.top * 8 + 15 & ~15) : 0, k_lds = list_bytes + wave * T * 32 * D, lds0 = (u32)(size_t)(__attribute__((address_space(3))) char*)lds;
    const u32 row_bytes = 2 * (u32)row_el, v_off = 4 * g * row_bytes + 2 * CPL * c;
    const KLane<D> kl(lane, row_bytes);
    float* const s_o = reinterpret_cast<float*>(lds + list_bytes);   // (where K was)
    float2* const s_ml = reinterpret_cast<float2*>(s_o + W * a.cols * (D + 4));
    const int units = ((count << sub_shift) + T - 1) / T, u0 = (int)((long)units * split / a.splits), u1 = (int)((long)units * (split + 1) / a.splits);

    for (int careful = 0;; ++careful) {
        float m = -inf, l = 0.0f;
        f32x4 o[CPL];
#pragma unroll
        for (int t = 0; t < CPL; ++t) o[t] = f32x4{0, 0, 0, 0};
        auto go = [&](auto is_careful) {
            constexpr bool CAREFUL = decltype(is_careful)::value;
            for (int u = u0 + wave; u < u1; u += W) {
                VTiles<D, T> f;
                int sees[T], tok[T];
                u32 place[T];
#pragma unroll
                for (int x = 0; x < T; ++x) {
                    const int sub = T * u + x, e = sub >> sub_shift, part = 16 * (sub & ((1 << sub_shift) - 1)), at = min(e, count - 1);
                    // (scalars: what a wave's branches go by, for a matrix instruction runs whatever the lanes' mask says)
                    u32 block;
                    if constexpr (LONG) { const uint2 ent = list[at]; block = __builtin_amdgcn_readfirstlane(ent.x); place[x] = __builtin_amdgcn_readfirstlane(ent.y) + part; }
                    else { block = __builtin_amdgcn_readlane(e_block, at); place[x] = __builtin_amdgcn_readlane(e_at, at) + part; }
                    tok[x] = e < count ? (int)block * a.block + part : n;             // (behind the list's end: nothing)
                    kl.fetch(reinterpret_cast<const char*>(kv + (size_t)place[x] * row_el), row_bytes, lds0 + k_lds + x * 32 * D, lane);
                }
#pragma unroll
                for (int x = 0; x < T; ++x) f.load(x, reinterpret_cast<const char*>(kv + (size_t)place[x] * row_el + v_el), row_bytes, v_off);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * T) : "memory");          // K is there (V, 4 T loads, came behind it)
                f32x4 s4[T];
#pragma unroll
                for (int x = 0; x < T; ++x) {
                    s4[x] = kl.template scores<F16>(lds + k_lds + x * 32 * D, [&](int s) { return q[s]; });
                    if (tok[x] >= n) s4[x] = f32x4{0, 0, 0, 0};      // (whatever lies behind the row's end: not worth the careful pass)
                    sees[x] = n - tok[x] - 4 * g;
                }
#pragma unroll
                for (int x = 0; x < T; ++x)
                    if (tok[x] + 16 > n) f.drop_v(x, n - tok[x], g);
                Terms<F16> b[T / 2];
                uint4 one[T / 2];
                weigh<F16, D, T, CAREFUL>(s4, sees, a.scale2, m, l, o, b, one);
#pragma unroll
                for (int y = 0; y < T / 2; ++y) weighted<F16, D, CAREFUL>([&](int t) { return f.vt(y, t); }, b[y], one[y], o);
            }
        };
        if (__builtin_expect(careful, 0)) go(std::true_type{});
        else go(std::false_type{});
        __syncthreads();                                             // (everyone's K has been read)
        put_columns<D>(s_o, s_ml, wave, a.cols, c, g, m, l, o);
        __syncthreads();
        bool bad = false;
        for (int it = tid; it < gh * (D / 4); it += 64 * W) {
            const int cc = it / (D / 4), d = it % (D / 4) * 4;
            float top, sum, acc[4];
            bad |= !merge_columns<D, W>(s_o, s_ml, a.cols, cc, d, top, sum, acc);
            const size_t row = (size_t)i * a.Hq + h * G + h0 + cc;
            if (a.splits > 1) {
                *reinterpret_cast<float4*>(a.part_o + (row * a.splits + split) * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (row * a.splits + split) * 2) = make_float2(top, count ? sum : -1.0f);      // (-1: the row lists nothing)
            } else store_columns<F16>(a.out + row * D + d, a.out_al, count != 0, sum, acc);
        }
        if (careful || !__builtin_amdgcn_readfirstlane(__syncthreads_or(bad))) break;
    }
}

// NC tiles of 16 columns whose rows share a request's blocks.  The waves of a block share the list's tokens, 32 in turn, each keeps all columns, and they meet in LDS
// at the end.
template <int F16, int D, int W, int NC>
__global__ __launch_bounds__(64 * W, 2) void k_block_attn_rows(BlockAttnArgs a) {
    constexpr int CPL = D / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int s_len[16], s_req[16], s_count[W], s_next, s_seen;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const float inf = __uint_as_float(0x7f800000u);
    // block -> (kv head, tile of rows), kv heads neighbours as above
    const int h = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv, G = a.Hq / a.Hkv, rpt = 16 / G;      // rpt: rows of a tile of columns
    const int i0 = tile * NC * rpt, R = min(NC * rpt, a.n_rows - i0);
    const int* const lists = a.blocks + ((size_t)i0 * a.Hkv + h) * a.top;
    if (tid < 16) {
        int len = 0, req = -1;
        if (tid < R) {
            len = a.q_kvlen[i0 + tid];
            req = a.q_req[i0 + tid];
            if (len <= 0 || req < 0 || req >= a.n_req || a.max_kvlen <= 0) { len = 0; req = -1; }
            len = min(len, a.max_kvlen);
        }
        s_len[tid] = len; s_req[tid] = req;
    }
    __syncthreads();
    const int rc = c / G, hc = c % G;                                // the column's row (of its tile) and head
    uint4 q[NC][D / 32];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const bool col = rc < rpt && n * rpt + rc < R;
        load_q<D>(q[n], a.q + (size_t)(i0 + (col ? n * rpt + rc : 0)) * a.q_stride + (size_t)(h * G + (col ? hc : 0)) * D + 8 * g, a.q_al, col, a.negate);
    }
    const int sub_shift = a.block == 16 ? 0 : a.block == 32 ? 1 : a.block == 64 ? 2 : 3, per = a.page_size / a.block;
    const size_t row_el = (size_t)a.Hkv * D, v_el = (size_t)a.page_size * row_el;      // elements between tokens, from K to V
    const bf16_t* const kv = a.kv + (size_t)h * D;
    const u32 row_bytes = 2 * (u32)row_el, v_off = 4 * g * row_bytes + 2 * CPL * c, k_lds = a.k_at + wave * 128 * D, lds0 = (u32)(size_t)(__attribute__((address_space(3))) char*)lds;
    const KLane<D> kl(lane, row_bytes);
    u32* const s_bits = reinterpret_cast<u32*>(lds);                 // two blocks' rows a word
    uint2* const list = reinterpret_cast<uint2*>(lds) + ATTN_WINDOW / 4;     // {block from the window's first << 16 | rows; its first token's place}
    float* const s_o = reinterpret_cast<float*>(lds);                // after the loops (where list and K were)
    float2* const s_ml = reinterpret_cast<float2*>(s_o + W * 16 * (D + 4));

    const int my_req = lane < R ? s_req[lane] : -1, my_len = lane < R ? s_len[lane] : 0;
    for (int ra = 0; ra < R;) {
        const int req = __builtin_amdgcn_readlane(my_req, ra);
        if (req < 0) { ++ra; continue; }
        const int p0 = a.indptr[req], np = a.indptr[req + 1] - p0;
        int n_most;
        const int rb = run_of(my_req, my_len, ra, R, lane, req, n_most);
        int own[NC];                                                 // tokens that the column's row sees
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int r = n * rpt + rc;
            own[n] = rc < rpt && r >= ra && r < rb ? s_len[r] : 0;
        }
        for (int careful = -1;;) {                                   // -1, then, if need be, the run's rows one by one
            float m[NC], l[NC];
            f32x4 o[NC][CPL];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                m[n] = -inf; l[n] = 0.0f;
#pragma unroll
                for (int t = 0; t < CPL; ++t) o[n][t] = f32x4{0, 0, 0, 0};
            }
            const int v_len = careful >= 0 ? __builtin_amdgcn_readlane(my_len, careful) : n_most;     // V of tokens from here on is taken as zero
            if (tid == 0) s_seen = 0;
            for (int w0 = 0; w0 >= 0;) {                             // windows of blocks
                for (int i = tid; i < ATTN_WINDOW / 2; i += 64 * W) s_bits[i] = 0;
                if (tid == 0) s_next = 0x7fffffff;
                __syncthreads();
                for (int r = ra + wave; r < rb; r += W) {
                    const int* const from = lists + (size_t)r * a.Hkv * a.top;
                    row_entries(from, first_entry(from, a.top, lane), a.top, (__builtin_amdgcn_readlane(my_len, r) - 1) / a.block + 1, lane, [&](int j, bool ok) {
                        if (!ok || j < w0) return;
                        if (j - w0 < ATTN_WINDOW) atomicOr(&s_bits[(j - w0) >> 1], 1u << (r + 16 * ((j - w0) & 1)));
                        else atomicMin(&s_next, j);
                    });
                }
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
                int at = upto - mine, count = 0;
                for (int x = 0; x < W; ++x) { if (x < wave) at += s_count[x]; count += s_count[x]; }
                count = __builtin_amdgcn_readfirstlane(count);
                for (int i = 0; mine && i < 2 * WPT; ++i) {
                    u32 rows = bits[0];
#pragma unroll
                    for (int x = 1; x < WPT; ++x) rows = i >> 1 == x ? bits[x] : rows;
                    rows = i & 1 ? rows >> 16 : rows & 0xffffu;
                    if (!rows) continue;
                    list[at++].x = (u32)(tid * WPT * 2 + i) << 16 | rows;
                }
                __syncthreads();
                u32 seen = 0;
                for (int e = tid; e < count; e += 64 * W) {          // their pages, a thread an entry
                    const u32 word = list[e].x;
                    const int j = w0 + (int)(word >> 16), pj = j / per;
                    int pg = pj < np ? a.indices[p0 + pj] : -1;
                    const bool ok = pg >= 0 && pg < a.n_pages;
                    pg = ok ? pg : 0;                                // (nobody's: page 0 is read and masked)
                    list[e] = make_uint2(ok ? word : word & 0xffff0000u, (u32)pg * 2 * a.page_size + (u32)(j - pj * per) * a.block);
                    seen |= ok ? word & 0xffffu : 0u;
                }
                if (seen) atomicOr(&s_seen, (int)seen);
                __syncthreads();
                const int tiles = count << sub_shift, units = (tiles + 1) / 2;
                u32 place[2];
                auto fetch = [&](int u, u32 to) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int sub = min(2 * u + x, tiles - 1);
                        place[x] = __builtin_amdgcn_readfirstlane(list[sub >> sub_shift].y) + 16 * (sub & ((1 << sub_shift) - 1));
                        kl.fetch(reinterpret_cast<const char*>(kv + (size_t)place[x] * row_el), row_bytes, to + x * 32 * D, lane);
                    }
                };
                auto go = [&](auto is_careful) {
                    constexpr bool CAREFUL = decltype(is_careful)::value;
                    u32 buf = 0;                                     // the wave's two K buffers in turn
                    fetch(wave, lds0 + k_lds);
                    for (int u = wave; u < units; u += W) {
                        dma_wait();                                  // (V of the unit before has been used: only this K is on its way)
                        VTiles<D, 2> f;
                        u32 rows[2];
                        int tok[2];
                        const u32 here[2] = {place[0], place[1]};
                        fetch(min(u + W, units - 1), lds0 + k_lds + (buf ^ 64 * D));      // (behind the last: asked for once more and not used)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int sub = min(2 * u + x, tiles - 1), e = sub >> sub_shift;
                            const u32 word = __builtin_amdgcn_readfirstlane(list[e].x);               // (scalars, as above)
                            rows[x] = 2 * u + x < tiles ? word & 0xffffu : 0u;                        // (the odd last tile of blocks of 16: nobody's)
                            tok[x] = (w0 + (int)(word >> 16)) * a.block + 16 * (sub & ((1 << sub_shift) - 1));
                            f.load(x, reinterpret_cast<const char*>(kv + (size_t)here[x] * row_el + v_el), row_bytes, v_off);
                        }
                        f32x4 s4[NC][2];
#pragma unroll
                        for (int n = 0; n < NC; ++n)
#pragma unroll
                            for (int x = 0; x < 2; ++x) s4[n][x] = kl.template scores<F16>(lds + k_lds + buf + x * 32 * D, [&](int s) { return q[n][s]; });
                        buf ^= 64 * D;
#pragma unroll
                        for (int x = 0; x < 2; ++x)                  // (whatever lies behind the rows' end: not worth the careful passes)
                            if (rows[x] == 0 || tok[x] >= n_most)
#pragma unroll
                                for (int n = 0; n < NC; ++n) s4[n][x] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int x = 0; x < 2; ++x) {                // V that nobody, or not the careful row, may see
                            const bool none = rows[x] == 0 || (CAREFUL && !(rows[x] >> careful & 1));
                            if (none || tok[x] + 16 > v_len) f.drop_v(x, none ? 0 : v_len - tok[x], g);
                        }
#pragma unroll
                        for (int n = 0; n < NC; ++n) {
                            if (NC > 1 && !((rows[0] | rows[1]) >> (n * rpt) & ((1u << rpt) - 1))) continue;      // no row of this tile lists these tokens
                            int sees[2];
#pragma unroll
                            for (int x = 0; x < 2; ++x) sees[x] = rows[x] >> (n * rpt + rc) & 1 ? own[n] - tok[x] - 4 * g : 0;
                            Terms<F16> b[1];
                            uint4 one[1];
                            weigh<F16, D, 2, CAREFUL>(s4[n], sees, a.scale2, m[n], l[n], o[n], b, one);
                            weighted<F16, D, CAREFUL>([&](int t) { return f.vt(0, t); }, b[0], one[0], o[n]);
                        }
                    }
                    dma_wait();                                      // (nothing may land in LDS that is used anew)
                };
                if (wave < units) {
                    if (__builtin_expect(careful < 0, 1)) go(std::false_type{});
                    else go(std::true_type{});
                }
                __syncthreads();                                     // (the list has been read)
                w0 = __builtin_amdgcn_readfirstlane(s_next);
                if (w0 == 0x7fffffff) w0 = -1;
                __syncthreads();
            }
            // the waves' shares of each column meet, a tile of columns at a time
            bool bad = false;
            const int seen_rows = s_seen;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                if (n) __syncthreads();
                put_columns<D>(s_o, s_ml, wave, 16, c, g, m[n], l[n], o[n]);
                __syncthreads();
                for (int it = tid; it < rpt * G * (D / 4); it += 64 * W) {
                    const int cc = it / (D / 4), d = it % (D / 4) * 4, r = n * rpt + cc / G;
                    if (r < ra || r >= rb || (careful >= 0 && r != careful)) continue;
                    float top, sum, acc[4];
                    bad |= !merge_columns<D, W>(s_o, s_ml, 16, cc, d, top, sum, acc);
                    store_columns<F16>(a.out + ((size_t)(i0 + r) * a.Hq + h * G + cc % G) * D + d, a.out_al, (seen_rows >> r & 1) != 0, sum, acc);
                }
            }
            const int again = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad));
            if (careful < 0 ? !again : careful + 1 >= rb) break;
            careful = careful < 0 ? ra : careful + 1;
        }
        ra = rb;
    }
}

// the splits of a row and head, a block of threads each: four channels a thread, the splits over the groups of D / 4 threads, all loads on their way at once (128 rows and heads
// of 32 splits: 3.9 us, 2.1 MB; a launch of nothing is 2)
template <int F16, int D>
__global__ __launch_bounds__(256) void k_block_attn_merge(BlockAttnArgs a) {
    constexpr int LPD = D / 4, GROUPS = 256 / LPD, MOST = 64 / GROUPS;
    __shared__ float s_o[GROUPS][D + 4];
    const int at = blockIdx.x, lane = threadIdx.x & 63, d = threadIdx.x % LPD * 4, grp = threadIdx.x / LPD;
    const float inf = __uint_as_float(0x7f800000u);
    const float2* const ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)at * a.splits;
    float4 o[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int z = grp + i * GROUPS;
        if (z < a.splits) o[i] = *reinterpret_cast<const float4*>(a.part_o + ((size_t)at * a.splits + z) * D + d);
    }
    const float2 mine = lane < a.splits ? ml[lane] : make_float2(-inf, 0.0f);
    const int i = at / a.Hq, len = min(a.q_kvlen[i], a.max_kvlen), req = a.q_req[i];
    if (len <= 0 || req < 0 || req >= a.n_req) return;               // (the whole block: its parts were not written either)
    float top = mine.x;
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float f = __builtin_amdgcn_exp2f(mine.x - (top == -inf ? 0.0f : top));
    const float sum = butterfly<64>(lane < a.splits ? f * mine.y : 0.0f);
    const bool none = __shfl(mine.y, 0, 64) == -1.0f;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int x = 0; x < MOST; ++x) {
        const int z = grp + x * GROUPS;
        const float w = __shfl(f, z & 63, 64);
        if (z < a.splits) { acc.x = __fmaf_rn(w, o[x].x, acc.x); acc.y = __fmaf_rn(w, o[x].y, acc.y); acc.z = __fmaf_rn(w, o[x].z, acc.z); acc.w = __fmaf_rn(w, o[x].w, acc.w); }
    }
    *reinterpret_cast<float4*>(&s_o[grp][d]) = acc;
    __syncthreads();
    if (threadIdx.x < D) {
        float all = 0.0f;
#pragma unroll
        for (int x = 0; x < GROUPS; ++x) all += s_o[x][threadIdx.x];
        a.out[(size_t)at * D + threadIdx.x] = none ? 0 : f_elem<F16>(all / sum);
    }
}

// ================================================================================================
// entry points
// ================================================================================================
// 16-channel pieces of a call from which on threads go through several heads.  us in a captured graph, a slot a head / eight slots a row, 32 + 16 heads of 128: 64 rows 3.5 / 4.6,
// 300 4.0 / 4.8, 700 (268800 pieces) 5.4 / 5.5, 1500 9.1 / 8.1, 4000 18.9 / 17.4; 16 + 16, 16384 rows 51.7 / 46.6.
#define APPEND_MANY (1 << 18)
#define BY_TYPE_AND_DIM(KERN, c) \
    ((c).dtype == VOX_DTYPE_F16 ? ((c).head_dim == 128 ? (const void*)KERN<1, 128> : (const void*)KERN<1, 64>) \
                                : ((c).head_dim == 128 ? (const void*)KERN<0, 128> : (const void*)KERN<0, 64>))

static int launch_bounds(hipStream_t st, const vox_block_cache& c, const int* page, const int* slot, int n_rows) {
    if (n_rows == 0) return VOX_OK;
    BoundsArgs b{(const bf16_t*)c.kv, c.bounds, c.steps, page, slot, n_rows, c.n_pages, c.page_size, c.block, c.kv_heads};
    return launch(BY_TYPE_AND_DIM(k_block_bounds, c), dim3((unsigned)(((int64_t)n_rows + 63) / 64), c.kv_heads), 256, 0, st, b);
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
    if (((int64_t)a->heads + 2 * c.kv_heads) * D > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "rope_append: %d heads of %d channels are 2^31 or more", a->heads, D);
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
    const bool with = vec && c.bounds && a->n_own == a->n_rows && (int64_t)a->n_rows * c.kv_heads < 0x7fffffff;      // the bounds in the same launch
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
// How a call's rows are laid out: rows a block of threads, waves, parts of a row's blocks (above 1: their scores go through the workspace).
struct SelectShape { int qt, W, splits, stride; };
static SelectShape select_shape(const vox_block_select_args* a) {
    const vox_block_rows& r = a->rows;
    const int most = (int)(((int64_t)r.max_kvlen + a->cache.block - 1) / a->cache.block);
    // rows a tile: 16 while their keys take half a CU's LDS, 8 while they take most of it (4096 blocks), else (and for rows of different requests) one; together only
    // where there are enough of them, the more the more channels a row has to bring to matrix rows first.  us in a captured graph, a row / 16 rows together, 256 blocks, for
    // 64, 128, 256 and 512 rows: 16 heads on 8 of 128 10.6 / 12.3, 13.6 / 12.8, 21 / 13, 37 / 13.3; 32 on 8 10 / 13.6, 12.5 / 13.7, 21.5 / 13.8, 37 / 14.3; 32 on 2 8.8 / 19.4,
    // 8.8 / 19.8, 10.3 / 19.9, 14.1 / 20; 8 on 8 of 64 9.7 / 11.3, 10.6 / 11.3, 15.2 / 11.4, 25.2 / 11.8.  Of other numbers of blocks, a call of the fewest rows that go together: 24 blocks
    // 11.0 / 11.4, 10.9 / 11.4, 13.5 / 17.1, 11.1 / 11.2 in the same order, 1000 24 / 16, 26 / 18, 46 / 24, 15.7 / 14.9, 3000 65 / 33, 84 / 33, 141 / 36, 32 / 23.
    const int G = r.heads / a->cache.kv_heads;
    const bool many = r.n_own > 0 && r.n_rows >= 2 * (int64_t)r.n_own && (int64_t)r.n_rows * a->cache.kv_heads >= 576 + G * a->cache.head_dim / 2;
    SelectShape s{many && most <= 1024 ? 16 : many && most <= 4096 ? 8 : 1, 8, 1, 0};
    s.stride = most + (s.qt > 1 ? SEL_PAD : 0);
    if (s.qt > 1) return s;
    // us in a captured graph, 4 / 8 / 16 waves a row: 32 rows of 512 blocks 14.0 / 13.6 / 15.9, 128 of 256 17.0 / 23.6 / 44, 64 of 1024 31.0 / 30.7 / 37.8, 64 of 1500 (dim 64) 30.4 / 26.9 /
    // 37.1, 32 of 4096 71 / 58.9 / 57.8; beyond that the keys leave no room for the bounds on their way, and 16 waves take them to registers.
    s.W = most <= 512 ? 4 : most <= 4096 ? 8 : 16;
    // One CU draws some 35 bytes a ns: a row's bounds over several CUs where there are CUs left and a row has more than 512 blocks.
    const int64_t pairs = (int64_t)r.n_rows * a->cache.kv_heads, z = pairs ? ATTN_CUS / pairs : 0, parts = (most + 255) / 256;
    if (most > 512 && z >= 2) s.splits = (int)(z < parts ? z : parts);
    return s;
}
int64_t vox_block_select_workspace_bytes(const vox_block_select_args* a) {
    if (check_select(a) != VOX_OK) return -1;
    const SelectShape s = select_shape(a);
    return s.splits > 1 ? (int64_t)a->rows.n_rows * a->cache.kv_heads * s.stride * 4 : 0;
}
int vox_block_select_form(const vox_block_select_args* a) {
    if (check_select(a) != VOX_OK) return 0;
    const SelectShape s = select_shape(a);
    return s.splits > 1 ? -s.splits : s.qt;
}
int vox_block_select(vox_ctx* ctx, void* stream, const vox_block_select_args* a) {
    (void)ctx;
    VOX_TRY(check_select(a));
    const vox_block_cache& c = a->cache;
    const vox_block_rows& r = a->rows;
    if (r.n_rows == 0) return VOX_OK;
    if (!a->q || !a->blocks || (size_t)a->q & 1) return vox_fail(VOX_ERR_INVALID, "block_select: an operand is NULL, or does not lie on its type");
    const SelectShape z = select_shape(a);
    const int per = c.page_size / c.block, qt = z.qt, W = z.W;
    const int64_t room = z.splits > 1 ? (int64_t)r.n_rows * c.kv_heads * z.stride * 4 : 0;
    if (room && (!a->workspace || (size_t)a->workspace & 15 || a->workspace_bytes < room))
        return vox_fail(VOX_ERR_INVALID, "block_select: a workspace of %lld bytes on 16, %lld are wanted", (long long)(a->workspace ? a->workspace_bytes : 0), (long long)room);
    const int words = z.splits == 1 && z.stride > c.head_dim ? z.stride : c.head_dim;
    const size_t lds = (size_t)qt * words * 4 + 15 & ~(size_t)15, tile = 32 * (size_t)c.head_dim;
    SelectArgs s{(const bf16_t*)a->q, c.bounds, c.steps, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (long)a->q_stride,
                 r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages, c.page_size, c.block, a->top, a->first, a->last, z.stride,
                 ((size_t)a->q & 15) == 0 && a->q_stride % 8 == 0, z.splits, (int)lds, (u32*)a->workspace, per > 1 ? (u32)((1ull << 32) / per + 1) : 0u};
    const int64_t grid = ((int64_t)r.n_rows + qt - 1) / qt * c.kv_heads * z.splits;
    if (grid > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "block_select: %d rows of %d kv heads are more than a launch holds", r.n_rows, c.kv_heads);
#define SELECT_OF(QT, W, SPLIT, NT) (c.dtype == VOX_DTYPE_F16 ? (c.head_dim == 128 ? (const void*)k_block_select<1, 128, QT, W, SPLIT, NT> : (const void*)k_block_select<1, 64, QT, W, SPLIT, NT>) \
                                                             : (c.head_dim == 128 ? (const void*)k_block_select<0, 128, QT, W, SPLIT, NT> : (const void*)k_block_select<0, 64, QT, W, SPLIT, NT>))
    if (z.splits > 1) {
        VOX_TRY(launch(SELECT_OF(1, 4, true, 2), dim3((unsigned)grid), 256, lds + 8 * tile, (hipStream_t)stream, s));
        return launch((const void*)k_block_choose<16>, dim3((unsigned)(grid / z.splits)), 1024, 0, (hipStream_t)stream, s);
    }
    if (qt == 16) return launch(SELECT_OF(16, 8, false, 1), dim3((unsigned)grid), 512, lds + 8 * tile, (hipStream_t)stream, s);
    if (qt == 8) return launch(SELECT_OF(8, 8, false, 0), dim3((unsigned)grid), 512, lds, (hipStream_t)stream, s);
    if (W == 8) return launch(SELECT_OF(1, 8, false, 2), dim3((unsigned)grid), 512, lds + 16 * tile, (hipStream_t)stream, s);
    return W == 4 ? launch(SELECT_OF(1, 4, false, 2), dim3((unsigned)grid), 256, lds + 8 * tile, (hipStream_t)stream, s)
                  : launch(SELECT_OF(1, 16, false, 0), dim3((unsigned)grid), 1024, lds, (hipStream_t)stream, s);
#undef SELECT_OF
}

static int check_attention(const vox_block_attention_args* a) {
    if (!a) return vox_fail(VOX_ERR_INVALID, "block_attention: no arguments");
    VOX_TRY(check_cache("block_attention", a->cache, true));
    VOX_TRY(check_rows("block_attention", a->cache, a->rows));
    if (a->top < 0 || a->top > VOX_BLOCK_TOP_MAX) return vox_fail(VOX_ERR_INVALID, "block_attention: lists of %d blocks (up to %d)", a->top, VOX_BLOCK_TOP_MAX);
    if (a->q_stride < 0) return vox_fail(VOX_ERR_INVALID, "block_attention: a stride is negative");
    if (!(fabsf(a->scale) <= 2e38f)) return vox_fail(VOX_ERR_INVALID, "block_attention: a scale of %g (finite, and so times log2 e)", (double)a->scale);
    return VOX_OK;
}
// How a call's rows are laid out: rows a tile, and the parts that a row's list is split into.
struct AttnShape { int tiles, per_tile, splits, head_tiles, W; };      // tiles of columns (0: a row a block of threads), rows a block, .., waves
static AttnShape attn_shape(const vox_block_attention_args* a, int cus) {
    const vox_block_rows& r = a->rows;
    const int G = r.heads / a->cache.kv_heads;
    AttnShape s{0, 1, 1, (G + 15) / 16, 8};
    // Rows together pay once there are enough of them: a tile's block of threads goes through what all its rows list, however few of them there are, a row's through its own list, 15 to
    // the us once the card is full; what R neighbouring rows list between them is some R^0.4 lists.  us, a row / rows together, lists of 2048 tokens, for 96, 128, 192 and 512 rows: 16 heads on
    // 8 of 128 59 / 80, 74 / 80, 104 / 79, 251 / 80; 32 on 8 52 / 58, 69 / 58, 98 / 59, 245 / 99; 8 on 8 of 64 39 / 55, 51 / 55, 74 / 56, 184 / 57; 14 on 2 of 64 (128 rows on) 18 / 35, 28 / 36,
    // 53 / 37; 32 on 2 of 128, 256 rows 39 / 42, 328 54 / 61, 420 69 / 60, 600 87 / 95, 900 136 / 116.  From lists of 64 tokens to ones of 8192 the crossings hold within a sixth: at the smallest number
    // of rows that goes together, 16 heads on 8 of 128 30 / 19 and 251 / 207, 32 on 8 24 / 18 and 196 / 154, 8 on 8 of 64 25 / 16 and 181 / 129, 32 on 2 20.5 / 18.6 and 149 / 175.
    // Eight waves a tile while that is a block of threads a CU, four where there are two (4 / 8 waves: 16 heads on 8, 512 rows 113 / 80, 1024 140 / 154; 8 on 8 of 64, 700 rows 97 / 102).
    if (r.n_own > 0 && r.n_rows >= 2 * (int64_t)r.n_own && G <= 16) {
        const int tiles = G > 1 ? 2 : 1, per_tile = tiles * (16 / G);
        const bool room = a->cache.head_dim == 64 || (int64_t)a->top * per_tile <= 2048;      // (eight waves' K at dim 128 are 128 of a CU's 160 KB, their lists 8 KB and 8 bytes an entry)
        const int waves = room && ((int64_t)r.n_rows + per_tile - 1) / per_tile * a->cache.kv_heads <= cus ? 8 : 4;
        const double pairs = waves == 8 ? 430.0 * pow(per_tile, 0.34) : 470.0 * pow(per_tile, 0.45);
        if ((double)r.n_rows * a->cache.kv_heads >= pairs) {
            s.tiles = tiles;
            s.per_tile = per_tile;
            s.W = waves;
            return s;
        }
    }
    const long tokens = (long)a->top * a->cache.block, blocks = (long)r.n_rows * a->cache.kv_heads * s.head_tiles;
    // A row's list over several blocks of threads, one for each CU that has none, 256 tokens at least; a second launch joins them (some 3 us of host time, so not for 1024
    // tokens, 11.4 / 9.4).  us in a captured graph, one block of threads a row / parts: 16 heads on 8 of 128, 1 row of 2048 tokens 19.4 / 10.2, 4 rows 25.8 / 16.7, 16 rows
    // 39.1 / 36.5; 32 on 2, 1 row of 4096 28.4 / 9.6, 4 rows of 8192 57 / 16.6, 16 rows 92 / 35 (two for each CU: 40); 32 on 8 of 64, 8 rows of 2048 21.2 / 16.9.
    if (tokens > 1024 && blocks > 0) {                               // (a call of no rows asks for its workspace too)
        const long z = (cus + blocks - 1) / blocks, most = (tokens + 255) / 256, parts = z < most ? z : most;
        s.splits = (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
    }
    return s;
}
int64_t vox_block_attention_workspace_bytes(const vox_block_attention_args* a) {
    if (check_attention(a) != VOX_OK) return -1;
    const AttnShape s = attn_shape(a, ATTN_CUS);
    return s.splits > 1 ? (int64_t)a->rows.n_rows * a->rows.heads * s.splits * (a->cache.head_dim + 2) * 4 : 0;
}
int vox_block_attention_form(const vox_block_attention_args* a) {
    if (check_attention(a) != VOX_OK) return 0;
    const AttnShape s = attn_shape(a, ATTN_CUS);
    return s.splits > 1 ? -s.splits : s.tiles ? s.per_tile : 1;
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
    const int64_t grid = ((int64_t)r.n_rows + z.per_tile - 1) / z.per_tile * z.splits * z.head_tiles * c.kv_heads;
    if (grid > 0x7fffffff) return vox_fail(VOX_ERR_INVALID, "block_attention: %d rows of %d heads are more than a launch holds", r.n_rows, r.heads);
    const bool one = z.tiles == 0;
    const float scale2 = fabsf(a->scale) * 1.44269504088896340736f;
    const int W = z.W, G = r.heads / c.kv_heads, cols = one && G < 16 ? G : 16;
    const bool big = a->top > 64;
    const size_t entries = (size_t)a->top * z.per_tile, merge = (size_t)W * cols * (c.head_dim + 4 + 2) * 4;
    const size_t lists = one ? (big ? ((size_t)a->top * 8 + 15 & ~(size_t)15) : 0) : ATTN_WINDOW * 2 + ((entries < ATTN_WINDOW ? entries : ATTN_WINDOW) * 8 + 15 & ~(size_t)15);
    const size_t keys = (size_t)W * 128 * c.head_dim, lds = one ? lists + (merge > keys ? merge : keys) : merge > lists + keys ? merge : lists + keys;
    BlockAttnArgs s{(const bf16_t*)a->q, (const bf16_t*)c.kv, r.q_req, r.q_kvlen, r.kv_indptr, r.kv_indices, a->blocks, (bf16_t*)a->out, (float*)a->workspace,
                    (float*)a->workspace + rows * c.head_dim, (long)a->q_stride, scale2 > LEAST_SCALE2 ? scale2 : LEAST_SCALE2, r.n_rows, r.n_req, r.heads, c.kv_heads, r.max_kvlen, c.n_pages,
                    c.page_size, c.block, a->top, z.splits, z.head_tiles, cols, ((size_t)a->q & 15) == 0 && a->q_stride % 8 == 0, ((size_t)a->out & 7) == 0, a->scale < 0.0f, (int)lists};
#define ATTN_OF(KERN, ...) (c.dtype == VOX_DTYPE_F16 ? (c.head_dim == 128 ? (const void*)KERN<1, 128, __VA_ARGS__> : (const void*)KERN<1, 64, __VA_ARGS__>) \
                                                     : (c.head_dim == 128 ? (const void*)KERN<0, 128, __VA_ARGS__> : (const void*)KERN<0, 64, __VA_ARGS__>))
    const void* kern = one ? (big ? ATTN_OF(k_block_attn_row, 8, true) : ATTN_OF(k_block_attn_row, 8, false))
                     : z.tiles == 2 ? (W == 8 ? ATTN_OF(k_block_attn_rows, 8, 2) : ATTN_OF(k_block_attn_rows, 4, 2)) : W == 8 ? ATTN_OF(k_block_attn_rows, 8, 1) : ATTN_OF(k_block_attn_rows, 4, 1);
#undef ATTN_OF
    VOX_TRY(launch(kern, dim3((unsigned)grid), 64 * W, lds, (hipStream_t)stream, s));
    if (z.splits == 1) return VOX_OK;
    return launch(BY_TYPE_AND_DIM(k_block_attn_merge, c), dim3((unsigned)(r.n_rows * r.heads)), 256, 0, (hipStream_t)stream, s);
}

}  // extern "C"
