// kv4_cache.cu -- tokens of the 4-bit paged key cache (attn_kv4.h) as contiguous bf16 K and V.
//
// Byte work: per element 2 bytes written and 17/32 read, no reuse. A thread turns 4 code bytes into 8 bf16
// elements, so a warp's store is 512 contiguous bytes and its load 128; each thread takes kUnroll tokens
// a block's stride apart, so that their loads are in flight together.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_kv4.h"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

extern "C" void ts_count_launch(void);

namespace ts {

namespace {

constexpr int kUnpackThreads = 256;
constexpr int kUnroll = 4;

// Block (x, y): a run of tokens of (sequence, kv head) y; blockIdx.z 0 for K, 1 for V.
template <int D>
__global__ void __launch_bounds__(kUnpackThreads) kv4_unpack_kernel(const ts_kv4_problem p) {
    constexpr int LANES = D / 8, TOKENS = kUnpackThreads / LANES;  // threads per token, tokens per pass
    pdl_wait();
    pdl_trigger();
    const uint8_t *codes = blockIdx.z ? p.v_codes : p.k_codes, *scales = blockIdx.z ? p.v_scales : p.k_scales;
    uint16_t *out = blockIdx.z ? p.V : p.K;
    const int e = threadIdx.x % LANES;
    for (long long y = blockIdx.y; y < (long long)p.B * p.Hkv; y += gridDim.y) {
        const int b = (int)(y / p.Hkv), h = (int)(y - (long long)b * p.Hkv);
        const int s0 = blockIdx.x * TOKENS * kUnroll + threadIdx.x / LANES;
        uint32_t c[kUnroll], sc[kUnroll];
        bool have[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int s = s0 + j * TOKENS;
            have[j] = s < p.S;
            int code = 0;
            if (have[j]) {
                const int pos = ld_plan(p.positions + (long long)b * p.S + s);
                const int lp = pos >= 0 ? pos / p.page_size : p.max_pages;
                int page = -1;
                if (lp < p.max_pages) {
                    page = ld_plan(p.block_table + (size_t)b * p.max_pages + lp);
                    if (page < 0 || page >= p.num_pages) code = kDevErrBadPage;
                } else {
                    code = kDevErrBadPos;
                }
                have[j] = code == 0;
                if (have[j]) {
                    const size_t row = ((size_t)page * p.Hkv + h) * p.page_size + (pos - lp * p.page_size);
                    c[j] = *reinterpret_cast<const uint32_t *>(codes + row * (D / 2) + 4 * e);
                    sc[j] = scales[row * (D / ATTN_KV4_GROUP) + e / (ATTN_KV4_GROUP / 8)];
                } else if (e == 0) {
                    atomicOr(p.status, code);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (!have[j]) continue;
            const __half_raw hr = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)sc[j], __NV_E4M3);
            const float f = __half2float(__half(hr));
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = (float)((int)((c[j] >> (8 * i)) & 15u) - 8), hi = (float)((int)((c[j] >> (8 * i + 4)) & 15u) - 8);
                w[i] = pack_bf16x2(lo * f, hi * f);
            }
            *reinterpret_cast<uint4 *>(out + ((size_t)y * p.S + s0 + j * TOKENS) * D + 8 * e) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

template <int D>
int launch_unpack(const ts_kv4_problem *P, cudaStream_t st) {
    constexpr int RUN = kUnpackThreads / (D / 8) * kUnroll;
    const long long y = (long long)P->B * P->Hkv;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)P->S + RUN - 1) / RUN), (unsigned)(y < 65535 ? y : 65535), 2);
    cfg.blockDim = dim3(kUnpackThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kv4_unpack_kernel<D>, *P) != cudaSuccess) return ATTN_ERR_CUDA;
    ts_count_launch();
    return ATTN_OK;
}

}  // namespace

}  // namespace ts

extern "C" int ts_launch_kv4_unpack(const ts_kv4_problem *P, void *stream) {
    if (P->B <= 0 || P->S <= 0) return ATTN_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return P->D == 64 ? ts::launch_unpack<64>(P, st) : ts::launch_unpack<128>(P, st);
}
