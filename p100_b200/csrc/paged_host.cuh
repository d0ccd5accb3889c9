// paged_host.cuh — what the translation units of the paged cache share on the
// host: the checks of the descriptor and the buffers, the workspace of the
// attention calls, the pages' tensor maps and the append's launch.
#pragma once
#include <algorithm>
#include <climits>
#include <cmath>

#include <cudaTypedefs.h>

#include "fa_paged.cuh"
#include "fa_paged_tc.cuh"
#include "paged_append.cuh"

namespace p100b {
namespace {

size_t round256(size_t x) { return (x + 255) & ~size_t(255); }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Dynamic shared memory beyond 48 KB, once per kernel and device.
template <typename K>
p100_status allow_smem(K kern, size_t bytes, int (&configured)[64], const char* what) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return cuda_status(e, what);
    if (configured[dev]) return P100_OK;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)))
        return cuda_status(e, what);
    configured[dev] = 1;
    return P100_OK;
}

// The descriptor with its defaults filled in, or the reason it is refused.
const char* paged_reason(const p100_paged_desc& in, paged::Desc& d) {
    if (in.n_seq < 0 || in.n_tokens < 0 || in.max_q < 0 || in.n_pages < 0 || in.max_pages < 0)
        return "counts must not be negative";
    if (in.n_seq > P100_PAGED_MAX_SEQ) return "n_seq exceeds P100_PAGED_MAX_SEQ";
    if (in.n_head_q <= 0 || in.n_head_kv <= 0 || in.page_size <= 0) return "all dimensions must be positive";
    if (in.n_head_q % in.n_head_kv) return "n_head_q must be divisible by n_head_kv";
    if (in.head_dim != 64 && in.head_dim != 128) return "head_dim must be 64 or 128";
    if (in.dtype != P100_F16 && in.dtype != P100_BF16) return "dtype must be P100_F16 or P100_BF16";
    if (!std::isfinite(in.scale)) return "scale must be finite";
    if (!std::isfinite(in.softcap) || in.softcap < 0.0f) return "softcap must be finite and non-negative";
    if (in.softcap > 1e15f) return "softcap must be at most 1e15";   // hidden scores are set to -1e18
    if ((long long)in.n_tokens * in.n_head_q > INT_MAX) return "n_tokens * n_head_q exceeds 2^31 - 1";
    if ((long long)in.max_pages * in.page_size > INT_MAX) return "max_pages * page_size exceeds 2^31 - 1";
    const long long D = in.head_dim;
    d.n_seq = in.n_seq;
    d.n_tokens = in.n_tokens;
    d.max_q = in.max_q ? std::min(in.max_q, in.n_tokens) : in.n_tokens;
    d.n_head_q = in.n_head_q;
    d.n_head_kv = in.n_head_kv;
    d.group = in.n_head_q / in.n_head_kv;
    d.page_size = in.page_size;
    d.n_pages = in.n_pages;
    d.max_pages = in.max_pages;
    d.causal = in.causal != 0;
    d.token_stride = in.token_stride ? in.token_stride : D;
    d.head_stride = in.head_stride ? in.head_stride : in.page_size * D;
    d.page_stride = in.page_stride ? in.page_stride : (long long)in.n_head_kv * in.page_size * D;
    d.q_stride = in.q_stride ? in.q_stride : in.n_head_q * D;
    d.o_stride = in.o_stride ? in.o_stride : in.n_head_q * D;
    for (long long s : {d.token_stride, d.head_stride, d.page_stride}) {
        if (s < D) return "page strides must be at least head_dim";
        if (s % 8) return "strides must be multiples of 8 elements";
    }
    for (long long s : {d.q_stride, d.o_stride}) {
        if (s < in.n_head_q * D) return "q and o strides must be at least n_head_q * head_dim";
        if (s % 8) return "strides must be multiples of 8 elements";
    }
    return nullptr;
}

// CTAs of the mma.sync kernel: two on every SM.
constexpr int kMmaCtas = 2;
static_assert(paged::kMaxSeq == P100_PAGED_MAX_SEQ, "lengths in shared memory");

// Units of a sequence's kv head are counted in 32 bits.
bool fa_paged_too_long(const paged::Desc& d, int rows, int keys, int over) {
    const double tiles = std::ceil(double(d.max_q) * d.group / rows);
    return tiles * (double(d.max_pages) * d.page_size / keys + 1 + over) >= 4294967295.0;
}

// Partials of all kernels share one place: their calls follow one another.
struct FaPagedWs {
    size_t tickets, o, ml, cuts, total;
};
constexpr size_t kCutBytes = 32;   // of the tree kernel's note on a cut row tile
size_t fa_paged_ticket_bytes(int sms) { return round256(size_t(sms) * kMmaCtas * 2 * sizeof(unsigned)); }
FaPagedWs fa_paged_ws(const p100_paged_desc& in, int sms) {
    const size_t rows = size_t(sms) * 2 * std::max(kMmaCtas * fap::kRows, fatc::kRows);
    FaPagedWs w;
    w.tickets = fa_paged_ticket_bytes(sms);   // first, so that init clears little
    w.o = round256(rows * in.head_dim * sizeof(float));
    w.ml = round256(rows * 2 * sizeof(float));
    w.cuts = round256(size_t(sms) * kCutBytes);
    w.total = w.tickets + w.o + w.ml + w.cuts;
    return w;
}

// The pages as a 4-d tensor (head_dim, token of the page, kv head, page) in
// boxes of 64 values x `box` tokens with the 128-byte swizzle.
p100_status page_map(CUtensorMap* map, const void* base, const p100_paged_desc& in, const paged::Desc& d, int box) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    if (!encode) return set_error(P100_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[4] = {cuuint64_t(in.head_dim), cuuint64_t(d.page_size), cuuint64_t(d.n_head_kv),
                                cuuint64_t(d.n_pages)};
    const cuuint64_t strides[3] = {cuuint64_t(d.token_stride) * 2, cuuint64_t(d.head_stride) * 2,
                                   cuuint64_t(d.page_stride) * 2};
    const cuuint32_t boxes[4] = {64, cuuint32_t(box), 1, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    const CUresult r =
        encode(map, in.dtype == P100_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
               const_cast<void*>(base), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return set_error(P100_ERR_INVALID, "page tensor map rejected (error %d): strides or extents", int(r));
    return P100_OK;
}

// The checks and parameters that the appends share: the descriptor, the fused
// rows, the norms and the buffers; `why` is the rotation's own refusal.  blocks
// stays 0 where there is nothing to do.
p100_status append_params(const p100_paged_desc* desc, const void* qkv, int qkv_type, long long qkv_stride,
                          const float* q_norm, const float* k_norm, float eps, const char* why, const int* block_table,
                          const int* q_start, const int* kv_len, void* q, void* k_pages, void* v_pages, int threads,
                          paged::AppendParams& prm, unsigned& blocks) {
    blocks = 0;
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    if (const char* bad = paged_reason(*desc, prm.d)) return set_error(P100_ERR_INVALID, "%s", bad);
    if (qkv_type != P100_F32 && qkv_type != P100_F16 && qkv_type != P100_BF16)
        return set_error(P100_ERR_INVALID, "unknown qkv type %d", qkv_type);
    const long long heads = (long long)desc->n_head_q + 2LL * desc->n_head_kv, width = heads * desc->head_dim;
    if (qkv_stride == 0) qkv_stride = width;
    if (qkv_stride < width) return set_error(P100_ERR_INVALID, "qkv_stride must be at least a fused row");
    if (qkv_stride * (qkv_type == P100_F32 ? 4 : 2) % 16)
        return set_error(P100_ERR_INVALID, "qkv rows must be 16-byte aligned");
    if ((q_norm || k_norm) && !(std::isfinite(eps) && eps >= 0.0f))
        return set_error(P100_ERR_INVALID, "eps must be finite and non-negative");
    if (why) return set_error(P100_ERR_INVALID, "%s", why);
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (desc->n_tokens == 0 || desc->n_seq == 0) return P100_OK;
    if (!qkv || !block_table || !q_start || !kv_len || !q || !k_pages || !v_pages)
        return set_error(P100_ERR_INVALID, "null buffer");
    if (!aligned(qkv, 16) || !aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
        return set_error(P100_ERR_INVALID, "qkv, q and the pages must be 16-byte aligned");
    prm.d.block_table = block_table;
    prm.d.q_start = q_start;
    prm.d.kv_len = kv_len;
    prm.qkv = qkv;
    prm.qkv_stride = qkv_stride;
    prm.q_norm = q_norm;
    prm.k_norm = k_norm;
    prm.eps = eps;
    prm.q = q;
    prm.k = k_pages;
    prm.v = v_pages;
    // as many warps a token as give every SM kAppendWarps of them, and no warp
    // more than kAppendMost steps
    const int at_once = qkv_type == P100_F32 ? 32 * paged::append_values<float>() / desc->head_dim
                                             : 32 * paged::append_values<__half>() / desc->head_dim;
    const int together = qkv_type == P100_F32 ? paged::append_steps<float>() : paged::append_steps<__half>();
    const long long steps = paged::Steps(desc->n_head_q, desc->n_head_kv, at_once).all();
    const long long fill = std::min((steps + together - 1) / together, (long long)sms * paged::kAppendWarps / desc->n_tokens);
    prm.warps = int(std::max({1LL, fill, (steps + paged::kAppendMost - 1) / paged::kAppendMost}));
    const long long all = ((long long)desc->n_tokens * prm.warps + threads / 32 - 1) / (threads / 32);
    if (all > INT_MAX) return set_error(P100_ERR_INVALID, "too many heads and tokens for one call");
    blocks = unsigned(all);
    return P100_OK;
}

// An append kernel for the call's types: launch<S, T, D>() is given them.
template <typename L>
p100_status append_typed(int qkv_type, int dtype, int head_dim, const L& launch) {
    auto to = [&](auto from) {
        using S = decltype(from);
        if (dtype == P100_F16)
            return head_dim == 64 ? launch.template operator()<S, __half, 64>() : launch.template operator()<S, __half, 128>();
        return head_dim == 64 ? launch.template operator()<S, __nv_bfloat16, 64>()
                              : launch.template operator()<S, __nv_bfloat16, 128>();
    };
    switch (qkv_type) {
        case P100_F32: return to(float());
        case P100_F16: return to(__half());
        default: return to(__nv_bfloat16());
    }
}

}  // namespace
}  // namespace p100b
