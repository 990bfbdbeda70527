// kv4_cache.cu -- writing and reading back the 4-bit paged key cache (attn_kv4.h): the QKV producer that
// appends to it, and its tokens as contiguous bf16 K and V. Byte work; HBM is the floor of both.
//
// Producer. A warp takes a token (or, when there are few, a part of its heads) and walks its q, k and v heads
// 32 / (D / 16) at a time, 16 elements a lane. The loads run four passes ahead through a ring in the warp's
// shared memory; what depends on the token alone (slot, cos and sin of the lane's frequencies) is loaded once a
// token. The arithmetic is attn_qkv_rope_paged_stream's, operation by operation, in packed fp32 pairs. It is
// bound by instruction issue: a variant of that call's kernel (bulk copies into a ring, a lane group per
// vector) ran 5,760 warp instructions a token of 32 + 2 * 8 heads of 128, this one 2,970; the norm and the
// rotation are template parameters, as branches of every pass they cost 10%. 16,384 such tokens: 75 to 79 us,
// 353 MB.
//
// A lane owns both members of each pair it rotates (rotate-half: elements [8i, 8i+8) and [rot/2 + 8i, +8);
// interleaved: 16 consecutive), as in qkv_rope.cu. A rotated key then crosses through the warp's shared
// memory, so that a lane holds 16 consecutive elements, half of a group, whatever the pairing was.
//
// Status. One extra CTA reads every position and page id of the call and stores the status word; the others
// skip what is out of range and report nothing. So no report can race with the clearing of an earlier
// call's, in a replayed graph either, and no memset sits between two calls.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "attn_kv4.h"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

extern "C" void ts_count_launch(void);

namespace ts {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;
constexpr int kDepth = 4;  // passes whose loads are in flight
constexpr unsigned kFull = 0xffffffffu;

// 16 bytes from global to shared memory, asynchronously; groups complete in the order of their commits.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Row of token position `pos` of sequence b in the pools' planes (page * Hkv, row in the page), or why not.
struct Slot {
    int page, row, code;
};
__device__ __forceinline__ Slot find_slot(const int *table, int b, int pos, int page_size, int max_pages, int num_pages) {
    Slot s{0, 0, 0};
    const int lp = pos >= 0 ? pos / page_size : max_pages;
    if (lp >= max_pages) {
        s.code = kDevErrBadPos;
        return s;
    }
    s.page = ld_plan(table + (size_t)b * max_pages + lp);
    s.row = pos - lp * page_size;
    if (s.page < 0 || s.page >= num_pages) s.code = kDevErrBadPage;
    return s;
}

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery's invariant divisor), for the loops in
// which d stays the same.
struct Divider {
    uint32_t m, shift;
    __device__ __forceinline__ explicit Divider(int d) {
        shift = d > 1 ? 32 - __clz(d - 1) : 0;
        m = (uint32_t)(((1ull << 32) * ((1ull << shift) - (uint32_t)d)) / (uint32_t)d) + 1u;
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> shift); }
};

// The status CTA: every token's slot is looked up and the codes of all are stored.
__device__ __forceinline__ void check_all(const int *positions, const int *table, int tokens, int S, int max_pos,
                                          int page_size, int max_pages, int num_pages, int *status) {
    // A warp takes runs of 32 * kFlight tokens, all loads of a run in flight together.
    const Divider by_page(page_size), by_seq(S);
    constexpr int kFlight = 16;
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    int code = 0;
    for (int t0 = (threadIdx.x >> 5) * 32 * kFlight; t0 < tokens; t0 += warps * 32 * kFlight) {
        int pos[kFlight], page[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const int t = t0 + 32 * j + lane;
            pos[j] = t < tokens ? ld_plan(positions + t) : 0;
        }
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const int t = t0 + 32 * j + lane, lp = pos[j] >= 0 ? by_page(pos[j]) : max_pages;
            page[j] = t < tokens && lp < max_pages ? ld_plan(table + (size_t)by_seq(t) * max_pages + lp) : 0;
            if (t < tokens && (lp >= max_pages || pos[j] >= max_pos)) code |= kDevErrBadPos;
        }
#pragma unroll
        for (int j = 0; j < kFlight; ++j)
            if (page[j] < 0 || page[j] >= num_pages) code |= kDevErrBadPage;
    }
    code = __syncthreads_or(code & kDevErrBadPos ? 1 : 0) * kDevErrBadPos |
           __syncthreads_or(code & kDevErrBadPage ? 1 : 0) * kDevErrBadPage;
    if (threadIdx.x == 0) *status = code;
}

__device__ __forceinline__ float2 unpack2(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float2 v) { return pack_bf16x2(v.x, v.y); }
// 16 consecutive bf16 elements, half of a group (the other half is the neighbouring lane's) -> nibbles and
// the group's scale s.
//
// The quotient x / s has to be rounded as the quotient, ties to even, and ties do occur (x has 8 bits, s has
// 4). y = x * (1/s) is off by at most one step of fp32; one correction by the exact residual x - y s (a step
// of Newton's iteration, as Markstein used it) lands on the tie when there is one, and never on one that is
// not there: next to a tie, x / s differs from it by 2^-12 at least. Adding 1.5 * 2^23 + 8 rounds it and leaves
// q + 8 in the low bits; eight of them, each times a power of 16, make a word once the constant's share is
// taken off. |x / s| <= 7.5, so nothing saturates, unless s is subnormal. Groups with a NaN, an infinity or a
// saturated scale take the plain way below.
__device__ __forceinline__ uint2 quantise(uint4 ra, uint4 rb, __nv_fp8_storage_t &s8) {
    const uint32_t r[8] = {ra.x, ra.y, ra.z, ra.w, rb.x, rb.y, rb.z, rb.w};
    uint32_t m2 = 0u;  // magnitudes order as their bits: largest of the even and of the odd elements
#pragma unroll
    for (int e = 0; e < 8; ++e) m2 = __vmaxu2(m2, r[e] & 0x7fff7fffu);
    uint32_t m = max(m2 & 0xffffu, m2 >> 16);
    m = max(m, __shfl_xor_sync(kFull, m, 1));
    uint32_t w[2];
    if (m < 0x4544u) {  // below 7 * 448
        s8 = __nv_cvt_float_to_fp8(__uint_as_float(m << 16) / 7.0f, __NV_SATFINITE, __NV_E4M3);
        const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw(s8, __NV_E4M3)));
        const float inv = s > 0.f ? 1.0f / s : 0.f;  // a scale of zero: every quotient is zero
        const float2 inv2 = make_float2(inv, inv), s2 = make_float2(-s, -s), magic = make_float2(12582920.f, 12582920.f);
        const bool small = s < 0.015625f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t t[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 x = unpack2(r[4 * h + e]);
                const float2 y = __fmul2_rn(x, inv2);
                float2 q = __ffma2_rn(__ffma2_rn(y, s2, x), inv2, y);
                if (small) q = make_float2(fminf(fmaxf(q.x, -8.f), 7.f), fminf(fmaxf(q.y, -8.f), 7.f));
                q = __fadd2_rn(q, magic);
                t[2 * e] = __float_as_uint(q.x), t[2 * e + 1] = __float_as_uint(q.y);
            }
            w[h] = t[7];
#pragma unroll
            for (int e = 6; e >= 0; --e) w[h] = w[h] * 16u + t[e];
            w[h] -= 0x4b400000u * 0x11111111u;
        }
    } else {
        float a = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 x = unpack2(r[e]);
            a = fmaxf(a, fmaxf(fabsf(x.x), fabsf(x.y)));  // (a NaN leaves a as it is)
        }
        // (both lanes of the group are here, other groups need not be)
        a = fmaxf(a, __shfl_xor_sync(3u << (threadIdx.x & 30), a, 1));
        s8 = __nv_cvt_float_to_fp8(a / 7.0f, __NV_SATFINITE, __NV_E4M3);
        const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw(s8, __NV_E4M3)));
        w[0] = w[1] = 0u;
        for (int e = 0; e < 16; ++e) {
            const uint32_t word = r[e >> 1];
            const float x = __uint_as_float((e & 1) ? word & 0xffff0000u : word << 16);
            const float q = s > 0.f ? x / s : 0.f;
            const uint32_t n = (uint32_t)((q == q ? (int)fminf(fmaxf(rintf(q), -8.f), 7.f) : 0) + 8) << (4 * (e & 7));
            if (e < 8)
                w[0] |= n;
            else
                w[1] |= n;
        }
    }
    return make_uint2(w[0], w[1]);
}

// |x| of the lower and the upper bf16 of a word as doubles, by moving bits: zero and subnormals come out below
// 2^-126, which a sum of squares does not see, infinities and NaN as 2^128 and more.
__device__ __forceinline__ double magnitude_lo(uint32_t w) {
    return __hiloint2double((int)((w & 0x7fffu) * 8192u + 0x38000000u), 0);
}
__device__ __forceinline__ double magnitude_hi(uint32_t w) {
    return __hiloint2double((int)(((w & 0x7fff0000u) >> 3) + 0x38000000u), 0);
}

// parts: how many items a token's head vectors are divided into. WHOLE: every element is rotated (rot == D).
// NORM: 1 q heads, 2 k heads, 3 both. zero: (-0, -0), see the rotation.
template <int D, bool NEOX, bool WHOLE, int NORM>
__global__ void __launch_bounds__(kAppendThreads, 3) kv4_append_kernel(const ts_rope_problem a, int parts, float2 zero) {
    constexpr int G = D / 16, VPW = 32 / G;  // lanes of a vector, vectors of a warp's pass
    __shared__ __align__(16) uint16_t cross[kAppendWarps][VPW * D];
    __shared__ __align__(16) float wq[D], wk[D];
    __shared__ __align__(16) uint8_t loads[kAppendWarps][kDepth * 1024];
    pdl_wait();
    pdl_trigger();
    const int tokens = a.B * a.S;
    if (blockIdx.x == 0) {  // (the first to start)
        check_all(a.positions, a.block_table, tokens, a.S, a.max_pos, a.page_size, a.max_pages, a.num_pages, a.status);
        return;
    }
    for (int e = threadIdx.x; e < D; e += blockDim.x) {
        if (NORM & 1) wq[e] = __uint_as_float((uint32_t)a.q_norm_w[e] << 16);
        if (NORM & 2) wk[e] = __uint_as_float((uint32_t)a.k_norm_w[e] << 16);
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane % G, grp = lane / G;
    // the lane's two runs of 8 elements
    const bool rot_lane = WHOLE || (NEOX ? li < (a.rot >> 4) : 16 * li < a.rot);
    const int oa = NEOX ? (rot_lane ? 8 * li : a.rot + 16 * (li - (a.rot >> 4))) : 16 * li;
    const int ob = NEOX && rot_lane ? (a.rot >> 1) + 8 * li : oa + 8;
    const int heads = a.Hq + 2 * a.Hkv, q_passes = (a.Hq + VPW - 1) / VPW, kv_passes = (a.Hkv + VPW - 1) / VPW;
    const int k_end = q_passes + kv_passes, passes = k_end + kv_passes, share = (passes + parts - 1) / parts;
    uint16_t *mine = cross[warp] + grp * D;
    // (parts > 1 only when there are few tokens: the items fit 32 bits)
    const unsigned items = (unsigned)tokens * (unsigned)parts, step = (gridDim.x - 1) * kAppendWarps;
    const unsigned item0 = (blockIdx.x - 1) * kAppendWarps + warp;
    auto token_of = [&](unsigned item) { return parts == 1 ? (int)item : (int)(item / (unsigned)parts); };
    // Loads run kDepth passes ahead of the arithmetic, over the ends of items: every lane copies its own 32
    // bytes of a pass into its own place of the warp's ring. A pass takes VPW heads of one kind (q, k, v). Where
    // the next load is: item, pass, head of this lane's group within its kind and how many the kind has, the
    // two runs' offsets in the token's row, passes left until the kind or the item changes.
    unsigned nitem = item0;
    int npass = 0, nlast = 0, nhead = 0, nheads = 0, na = 0, nb = 0, nleft = 0;
    const uint16_t *nsrc = a.qkv;
    auto seek = [&]() {
        const int kind = npass < q_passes ? 0 : (npass < k_end ? 1 : 2);
        const int from = kind == 0 ? 0 : (kind == 1 ? q_passes : k_end);
        nhead = (npass - from) * VPW + grp;
        nheads = kind == 0 ? a.Hq : a.Hkv;
        const int off = (nhead + (kind == 0 ? 0 : (kind == 1 ? a.Hq : a.Hq + a.Hkv))) * D;
        // (a value row is not rotated: 16 consecutive elements, as the quantiser wants them)
        na = off + (kind == 2 ? 16 * li : oa);
        nb = off + (kind == 2 ? 16 * li + 8 : ob);
        const int end = min(nlast, kind == 0 ? q_passes : (kind == 1 ? k_end : passes));
        nleft = end - npass;
        npass = end;  // (the pass after the run)
    };
    auto next_run = [&]() {  // the next run of passes of one kind; an item without a pass is stepped over
        if (npass >= nlast) {
            for (nitem += nlast > 0 ? step : 0; nitem < items; nitem += step) {
                const int tok = token_of(nitem);
                npass = (int)(nitem - (unsigned)tok * parts) * share;
                nlast = min(passes, npass + share);
                nsrc = a.qkv + (long long)tok * heads * D;
                if (npass < nlast) break;
            }
            if (nitem >= items) {
                nleft = 0x7fffffff;
                nheads = 0;  // nothing more is loaded
                return;
            }
        }
        seek();
    };
    const uint32_t ring = smem_u32(loads[warp]) + lane * 16;
    auto fetch = [&](int stage) {
        if (nhead < nheads) {
            copy16(ring + stage * 1024, nsrc + na);
            copy16(ring + stage * 1024 + 512, nsrc + nb);
        }
        copy_commit();
        if (--nleft == 0) {
            next_run();
        } else {
            nhead += VPW;
            na += VPW * D;
            nb += VPW * D;
        }
    };
    next_run();
    for (int st = 0; st < kDepth; ++st) fetch(st);
    int stage = 0;
    auto take = [&](uint4 &ra, uint4 &rb) {  // this pass's elements; its place takes the load kDepth passes on
        copy_wait<kDepth - 1>();
        ra = *reinterpret_cast<const uint4 *>(loads[warp] + stage * 1024 + lane * 16);
        rb = *reinterpret_cast<const uint4 *>(loads[warp] + stage * 1024 + lane * 16 + 512);
        fetch(stage);
        stage = (stage + 1) % kDepth;
    };
    float2 c[4], sn[4];
    // One pass over rotated heads (keys or queries): normed, rotated, rounded to bf16.
    auto rotated = [&](auto key_tag, uint4 ra, uint4 rb, uint4 &oa4, uint4 &ob4) {
        constexpr bool kKey = decltype(key_tag)::value;
        float2 x[8] = {unpack2(ra.x), unpack2(ra.y), unpack2(ra.z), unpack2(ra.w),
                       unpack2(rb.x), unpack2(rb.y), unpack2(rb.z), unpack2(rb.w)};
        if constexpr ((NORM & (kKey ? 2 : 1)) != 0) {
            float root;
            if (kKey) {
                // A last bit of the root can move a code by one: the k heads' sum is taken in double and the
                // root rounded once, whatever the order.
                const uint32_t w[8] = {ra.x, ra.y, ra.z, ra.w, rb.x, rb.y, rb.z, rb.w};
                double sd = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double u = magnitude_lo(w[e]), v = magnitude_hi(w[e]);
                    sd = fma(v, v, fma(u, u, sd));
                }
#pragma unroll
                for (int o = G / 2; o >= 1; o >>= 1) sd += __shfl_xor_sync(kFull, sd, o, G);
                // 1 / sqrt(v): the fp32 root, and one step of Newton's iteration in double
                const double v = sd * (1.0 / D) + (double)a.eps;
                const double r0 = (double)rsqrtf((float)v);
                const double r1 = fma(0.5 * r0, fma(-v * r0, r0, 1.0), r0);
                root = v > 1e-30 && v < 1e30 ? (float)r1 : (float)rsqrt(v);
                // An infinity or a NaN stands in the sum as a number of 2^256 and more. The root over an infinity is
                // zero, over a NaN it is one.
                if (__any_sync(kFull, !(v < 1e30))) {
                    uint32_t m = 0u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = __vmaxu2(m, w[e] & 0x7fff7fffu);
                    m = max(m & 0xffffu, m >> 16);
#pragma unroll
                    for (int o = G / 2; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o, G));
                    if (m >= 0x7f80u) root = m > 0x7f80u ? __uint_as_float(0x7fc00000u) : 0.f;
                }
            } else {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(x[e].y, x[e].y, fmaf(x[e].x, x[e].x, ss));
#pragma unroll
                for (int o = G / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o, G);
                root = rsqrtf(__fmaf_rn(ss, 1.0f / (float)D, a.eps));
            }
            const float *w = kKey ? wk : wq;
            const float2 r2 = make_float2(root, root);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float4 u = *reinterpret_cast<const float4 *>(w + oa + 2 * e);
                const float4 v = *reinterpret_cast<const float4 *>(w + ob + 2 * e);
                x[e] = __fmul2_rn(__fmul2_rn(x[e], r2), make_float2(u.x, u.y));
                x[e + 1] = __fmul2_rn(__fmul2_rn(x[e + 1], r2), make_float2(u.z, u.w));
                x[4 + e] = __fmul2_rn(__fmul2_rn(x[4 + e], r2), make_float2(v.x, v.y));
                x[5 + e] = __fmul2_rn(__fmul2_rn(x[5 + e], r2), make_float2(v.z, v.w));
            }
        }
        if (rot_lane) {
            // Each product is rounded, then their sum: products as FMAs with a zero that the compiler does not
            // know (it would fuse a packed product with the packed sum after it, whatever the intrinsics say),
            // differences as FMAs by -1.
            const float2 minus = make_float2(-1.f, -1.f);
            if (NEOX) {  // pairs (x[e], x[4 + e]) at frequencies 8 li + 2e, + 1
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 u = x[e], w = x[4 + e];
                    x[e] = __ffma2_rn(__ffma2_rn(w, sn[e], zero), minus, __ffma2_rn(u, c[e], zero));
                    x[4 + e] = __fadd2_rn(__ffma2_rn(w, c[e], zero), __ffma2_rn(u, sn[e], zero));
                }
            } else {  // pairs (x[e].x, x[e].y) at frequency 8 li + e
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = x[e].x, w = x[e].y;
                    const float cf = (e & 1) ? c[e >> 1].y : c[e >> 1].x, sf = (e & 1) ? sn[e >> 1].y : sn[e >> 1].x;
                    x[e].x = __fsub_rn(__fmul_rn(u, cf), __fmul_rn(w, sf));
                    x[e].y = __fadd_rn(__fmul_rn(w, cf), __fmul_rn(u, sf));
                }
            }
        }
        oa4 = make_uint4(pack2(x[0]), pack2(x[1]), pack2(x[2]), pack2(x[3]));
        ob4 = make_uint4(pack2(x[4]), pack2(x[5]), pack2(x[6]), pack2(x[7]));
    };
    for (unsigned item = item0; item < items; item += step) {
        const int tok = token_of(item), first = (int)(item - (unsigned)tok * parts) * share, last = min(passes, first + share);
        if (first >= last) continue;
        const int pos = ld_plan(a.positions + tok);
        const int b = tok / a.S, sq = tok - b * a.S;
        const Slot slot = find_slot(a.block_table, b, pos, a.page_size, a.max_pages, a.num_pages);
        uint4 ra, rb, oa4, ob4;
        if (slot.code != 0 || pos >= a.max_pos) {  // skipped whole (the status CTA reports it)
            for (int pass = first; pass < last; ++pass) take(ra, rb);
            continue;
        }
        if (rot_lane) {
            const float *row = a.cos_sin + (long long)pos * a.rot + 8 * li, *srow = row + (a.rot >> 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 cv = *reinterpret_cast<const float4 *>(row + 4 * i);
                const float4 sv = *reinterpret_cast<const float4 *>(srow + 4 * i);
                c[2 * i] = make_float2(cv.x, cv.y), c[2 * i + 1] = make_float2(cv.z, cv.w);
                sn[2 * i] = make_float2(sv.x, sv.y), sn[2 * i + 1] = make_float2(sv.z, sv.w);
            }
        }
        int pass = first;
        if (pass < q_passes) {
            int h = pass * VPW + grp;
            uint16_t *at = a.Q + (((long long)b * a.Hq + h) * a.S + sq) * D;
            const long long at_step = (long long)VPW * a.S * D;
            for (const int end = min(last, q_passes); pass < end; ++pass, h += VPW, at += at_step) {
                take(ra, rb);
                rotated(std::false_type{}, ra, rb, oa4, ob4);
                if (h < a.Hq) {
                    *reinterpret_cast<uint4 *>(at + oa) = oa4;
                    *reinterpret_cast<uint4 *>(at + ob) = ob4;
                }
            }
        }
        const long long row0 = (long long)slot.page * a.Hkv * a.page_size + slot.row;
        auto store = [&](uint4 x, uint4 y, int h, uint8_t *codes, uint8_t *scales) {
            __nv_fp8_storage_t s8;
            const uint2 w = quantise(x, y, s8);
            if (h < a.Hkv) {
                const long long row = row0 + (long long)h * a.page_size;
                *reinterpret_cast<uint2 *>(codes + row * (D / 2) + 8 * li) = w;
                if ((li & 1) == 0) scales[row * (D / ATTN_KV4_GROUP) + (li >> 1)] = s8;
            }
        };
        for (const int end = min(last, k_end); pass < end; ++pass) {
            take(ra, rb);
            rotated(std::true_type{}, ra, rb, oa4, ob4);
            *reinterpret_cast<uint4 *>(mine + oa) = oa4;
            *reinterpret_cast<uint4 *>(mine + ob) = ob4;
            __syncwarp();
            ra = *reinterpret_cast<const uint4 *>(mine + 16 * li);
            rb = *reinterpret_cast<const uint4 *>(mine + 16 * li + 8);
            __syncwarp();
            store(ra, rb, (pass - q_passes) * VPW + grp, a.k_codes, a.k_scales);
        }
        for (; pass < last; ++pass) {
            take(ra, rb);
            store(ra, rb, (pass - k_end) * VPW + grp, a.v_codes, a.v_scales);
        }
    }
}

// ---------------------------------------------------------------- reading back
// A thread turns 4 code bytes of a key and of a value into 8 bf16 elements each, so a warp's store is 512
// contiguous bytes. (n - 8) * s = (128 + n) * s - 136 * s in one bf16 FMA, exact: 128 + n is the bf16 number
// whose bits are 0x4300 + n, s has 4 significant bits, and 136 * s = 17 * s * 8 has at most 8.
constexpr int kUnpackThreads = 256;
constexpr int kUnroll = 4;  // heads whose loads are in flight together

__device__ __forceinline__ uint4 values8(uint32_t c, uint32_t s8) {
    const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)s8, __NV_E4M3);
    const float f = __half2float(__half(hr));
    const __nv_bfloat162 s = __float2bfloat162_rn(f), off = __float2bfloat162_rn(-136.f * f);
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // nibbles (i, i + 4)
        uint32_t v = ((c >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162 *>(&v), s, off);
        p[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
    return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632),
                      __byte_perm(p[2], p[3], 0x7632));
}

// Block (x, y): a run of tokens (of all sequences) and a share of the kv heads; what depends on the token
// alone is found once. Block (0, 0) stores the status.
template <int D>
__global__ void __launch_bounds__(kUnpackThreads) kv4_unpack_kernel(const ts_kv4_problem p, int heads_each) {
    constexpr int LANES = D / 8, TOKENS = kUnpackThreads / LANES;  // threads per token, tokens of a block
    pdl_wait();
    pdl_trigger();
    const int tokens = p.B * p.S;
    if (blockIdx.x == 0) {
        if (blockIdx.y == 0)
            check_all(p.positions, p.block_table, tokens, p.S, 0x7fffffff, p.page_size, p.max_pages, p.num_pages, p.status);
        return;
    }
    const int e = threadIdx.x % LANES;
    const int tok = (blockIdx.x - 1) * TOKENS + threadIdx.x / LANES;
    if (tok >= tokens) return;
    const int pos = ld_plan(p.positions + tok);
    const int b = tok / p.S, s = tok - b * p.S;
    const Slot slot = find_slot(p.block_table, b, pos, p.page_size, p.max_pages, p.num_pages);
    if (slot.code != 0) return;
    const int h0 = blockIdx.y * heads_each, h1 = min(p.Hkv, h0 + heads_each);
    const size_t row = ((size_t)slot.page * p.Hkv + h0) * p.page_size + slot.row;
    const uint8_t *kc = p.k_codes + row * (D / 2) + 4 * e, *vc = p.v_codes + row * (D / 2) + 4 * e;
    const uint8_t *ks = p.k_scales + row * (D / ATTN_KV4_GROUP) + e / (ATTN_KV4_GROUP / 8);
    const uint8_t *vs = p.v_scales + row * (D / ATTN_KV4_GROUP) + e / (ATTN_KV4_GROUP / 8);
    const size_t at = (((size_t)b * p.Hkv + h0) * p.S + s) * D + 8 * e;
    uint16_t *ko = p.K + at, *vo = p.V + at;
    const size_t code_step = (size_t)p.page_size * (D / 2), scale_step = (size_t)p.page_size * (D / ATTN_KV4_GROUP);
    const size_t out_step = (size_t)p.S * D;
    for (int h = h0; h < h1; h += kUnroll) {
        uint32_t k[kUnroll], v[kUnroll], sk[kUnroll], sv[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (h + j >= h1) break;
            k[j] = *reinterpret_cast<const uint32_t *>(kc + j * code_step);
            v[j] = *reinterpret_cast<const uint32_t *>(vc + j * code_step);
            sk[j] = ks[j * scale_step];
            sv[j] = vs[j * scale_step];
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (h + j >= h1) break;
            *reinterpret_cast<uint4 *>(ko + j * out_step) = values8(k[j], sk[j]);
            *reinterpret_cast<uint4 *>(vo + j * out_step) = values8(v[j], sv[j]);
        }
        kc += kUnroll * code_step, vc += kUnroll * code_step;
        ks += kUnroll * scale_step, vs += kUnroll * scale_step;
        ko += kUnroll * out_step, vo += kUnroll * out_step;
    }
}

template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, int threads, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...) != cudaSuccess) return ATTN_ERR_CUDA;
    ts_count_launch();
    return ATTN_OK;
}

template <int D, bool NEOX, bool WHOLE, int NORM>
int launch_append(const ts_rope_problem *P, cudaStream_t st) {
    constexpr int VPW = 32 / (D / 16);
    const long long tokens = (long long)P->B * P->S, wave = (long long)ts_num_sms() * 3 * kAppendWarps;
    const int passes = (P->Hq + VPW - 1) / VPW + 2 * ((P->Hkv + VPW - 1) / VPW);
    // few tokens: their heads are divided, down to one pass an item, to fill the GPU
    long long parts = (wave + tokens - 1) / tokens;
    if (parts > passes) parts = passes;
    const long long ctas = (tokens * parts + kAppendWarps - 1) / kAppendWarps, most = (long long)ts_num_sms() * 3;
    return launch(kv4_append_kernel<D, NEOX, WHOLE, NORM>, dim3((unsigned)((ctas < most ? ctas : most) + 1)), kAppendThreads,
                  st, *P, (int)parts, make_float2(-0.f, -0.f));
}

template <int D, bool NEOX, bool WHOLE>
int launch_append(const ts_rope_problem *P, cudaStream_t st) {
    switch ((P->q_norm_w ? 1 : 0) + (P->k_norm_w ? 2 : 0)) {
    case 0: return launch_append<D, NEOX, WHOLE, 0>(P, st);
    case 1: return launch_append<D, NEOX, WHOLE, 1>(P, st);
    case 2: return launch_append<D, NEOX, WHOLE, 2>(P, st);
    default: return launch_append<D, NEOX, WHOLE, 3>(P, st);
    }
}

template <int D>
int launch_append(const ts_rope_problem *P, cudaStream_t st) {
    const bool neox = P->style == ATTN_ROPE_NEOX, whole = P->rot == D;
    if (neox) return whole ? launch_append<D, true, true>(P, st) : launch_append<D, true, false>(P, st);
    return whole ? launch_append<D, false, true>(P, st) : launch_append<D, false, false>(P, st);
}

template <int D>
int launch_unpack(const ts_kv4_problem *P, cudaStream_t st) {
    constexpr int TOKENS = kUnpackThreads / (D / 8);
    const long long x = ((long long)P->B * P->S + TOKENS - 1) / TOKENS, wave = (long long)ts_num_sms() * 8;
    // few tokens: the heads are divided among blocks
    long long y = (wave + x - 1) / x;
    if (y > P->Hkv) y = P->Hkv;
    if (y > 65535) y = 65535;
    const int each = (int)((P->Hkv + y - 1) / y);
    return launch(kv4_unpack_kernel<D>, dim3((unsigned)(x + 1), (unsigned)((P->Hkv + each - 1) / each)), kUnpackThreads, st,
                  *P, each);
}

}  // namespace

}  // namespace ts

extern "C" int ts_launch_kv4_append(const ts_rope_problem *P, void *stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return P->D == 64 ? ts::launch_append<64>(P, st) : ts::launch_append<128>(P, st);
}

extern "C" int ts_launch_kv4_unpack(const ts_kv4_problem *P, void *stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return P->D == 64 ? ts::launch_unpack<64>(P, st) : ts::launch_unpack<128>(P, st);
}
