// serve.cu — the extern "C" entry points of include/p100/b200.h for prompts
// and batches: the append of new tokens to a paged cache, attention over it,
// and the scoring of logits.  A translation unit of its own, with its own
// g_device_error word, which p100_device_error reads through
// serve_device_error.
#include <climits>
#include <cmath>
#include <cstring>
#include <algorithm>

#include <cudaTypedefs.h>

#include "common.cuh"
#include "fa_paged.cuh"
#include "fa_paged_tc.cuh"
#include "logprobs.cuh"
#include "paged_append.cuh"

namespace p100b {

p100_status serve_device_error(int clear, int* value) {
    if (p100_status st = cuda_status(cudaMemcpyFromSymbol(value, g_device_error, sizeof *value), "read device flag"))
        return st;
    if (clear && *value) {
        const int zero = 0;
        return cuda_status(cudaMemcpyToSymbol(g_device_error, &zero, sizeof zero), "clear device flag");
    }
    return P100_OK;
}

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

// ------------------------------------------------------------ paged cache
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

// The tensor-core kernel takes calls in which a sequence may have more rows
// (new tokens x query heads per kv head) than the mma.sync kernel's row tile.
// One token each of 64 sequences of 8192 (64 / 8 heads): 245 us on the mma.sync
// kernel, 396 on the other; of 16 sequences (12 / 4 heads of 64) 31 and 59.
bool fa_paged_on_tc(const paged::Desc& d) { return (long long)d.max_q * d.group > fap::kRows && d.n_pages > 0; }

// Units of a sequence's kv head are counted in 32 bits.
bool fa_paged_too_long(const paged::Desc& d, int rows, int keys, int over) {
    const double tiles = std::ceil(double(d.max_q) * d.group / rows);
    return tiles * (double(d.max_pages) * d.page_size / keys + 1 + over) >= 4294967295.0;
}

// Partials of both kernels share one place: their calls follow one another.
struct FaPagedWs {
    size_t tickets, o, ml, total;
};
size_t fa_paged_ticket_bytes(int sms) { return round256(size_t(sms) * kMmaCtas * 2 * sizeof(unsigned)); }
FaPagedWs fa_paged_ws(const p100_paged_desc& in, int sms) {
    const size_t rows = size_t(sms) * 2 * std::max(kMmaCtas * fap::kRows, fatc::kRows);
    FaPagedWs w;
    w.tickets = fa_paged_ticket_bytes(sms);   // first, so that init clears little
    w.o = round256(rows * in.head_dim * sizeof(float));
    w.ml = round256(rows * 2 * sizeof(float));
    w.total = w.tickets + w.o + w.ml;
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

template <typename T, int D, bool CAP>
p100_status launch_fa_paged_tc(const fatc::Params& prm, const CUtensorMap& tmk, const CUtensorMap& tmv, int sms,
                               cudaStream_t stream) {
    static thread_local int configured[64] = {};
    auto kern = fatc::fa_paged_tc_kernel<T, D, CAP>;
    constexpr size_t fixed = fatc::smem_bytes<D>();
    if (p100_status st = allow_smem(kern, fixed + paged::Lengths::bytes(paged::kMaxSeq), configured,
                                    "cudaFuncSetAttribute(fa_paged_tc)"))
        return st;
    kern<<<sms, fatc::kThreads, fixed + paged::Lengths::bytes(prm.d.n_seq), stream>>>(prm, tmk, tmv);
    return cuda_status(cudaGetLastError(), "fa_paged_tc_kernel launch");
}
template <typename T>
p100_status launch_fa_paged_tc_d(const fatc::Params& prm, int head_dim, const CUtensorMap& tmk, const CUtensorMap& tmv,
                                 int sms, cudaStream_t s) {
    const bool cap = prm.softcap != 0.0f;
    if (head_dim == 64)
        return cap ? launch_fa_paged_tc<T, 64, true>(prm, tmk, tmv, sms, s)
                   : launch_fa_paged_tc<T, 64, false>(prm, tmk, tmv, sms, s);
    return cap ? launch_fa_paged_tc<T, 128, true>(prm, tmk, tmv, sms, s)
               : launch_fa_paged_tc<T, 128, false>(prm, tmk, tmv, sms, s);
}

template <typename T, int D, bool SPARE>
p100_status launch_fa_paged_mma(const fap::Params& prm, int sms, cudaStream_t stream) {
    static thread_local int configured[64] = {};
    auto kern = fap::fa_paged_kernel<T, D, SPARE>;
    constexpr size_t fixed = fap::smem_bytes<D>();
    if (p100_status st = allow_smem(kern, fixed + paged::Lengths::bytes(paged::kMaxSeq), configured,
                                    "cudaFuncSetAttribute(fa_paged)"))
        return st;
    kern<<<sms * kMmaCtas, fap::kThreads, fixed + paged::Lengths::bytes(prm.d.n_seq), stream>>>(prm);
    return cuda_status(cudaGetLastError(), "fa_paged_kernel launch");
}

template <typename T>
p100_status launch_fa_paged_mma_d(const fap::Params& prm, int head_dim, int sms, cudaStream_t s) {
    // 8 rows a kv head or fewer: the second parts of their probabilities take the other 8
    const bool spare = (long long)prm.d.max_q * prm.d.group <= fap::kRows / 2;
    if (head_dim == 64)
        return spare ? launch_fa_paged_mma<T, 64, true>(prm, sms, s) : launch_fa_paged_mma<T, 64, false>(prm, sms, s);
    return spare ? launch_fa_paged_mma<T, 128, true>(prm, sms, s) : launch_fa_paged_mma<T, 128, false>(prm, sms, s);
}

template <typename S, typename T>
p100_status launch_append(const paged::AppendParams& prm, int head_dim, unsigned blocks, cudaStream_t stream) {
    if (head_dim == 64)
        paged::paged_append_kernel<S, T, 64><<<blocks, paged::kAppendThreads, 0, stream>>>(prm);
    else
        paged::paged_append_kernel<S, T, 128><<<blocks, paged::kAppendThreads, 0, stream>>>(prm);
    return cuda_status(cudaGetLastError(), "paged_append_kernel launch");
}
template <typename S>
p100_status launch_append_to(const paged::AppendParams& prm, int dtype, int head_dim, unsigned blocks, cudaStream_t s) {
    return dtype == P100_F16 ? launch_append<S, __half>(prm, head_dim, blocks, s)
                             : launch_append<S, __nv_bfloat16>(prm, head_dim, blocks, s);
}

// ------------------------------------------------------------ logits
size_t dtype_bytes(int t) { return t == P100_F32 ? 4 : 2; }
const char* logprobs_reason(int rows, int n, int dtype, int top_k) {
    if (rows < 0 || n <= 0) return "rows must not be negative and n must be positive";
    if (n > lp::kMaxLogits) return "n exceeds 2^24";
    if (dtype != P100_F32 && dtype != P100_F16 && dtype != P100_BF16) return "unknown logit type";
    if (top_k < 0 || top_k > lp::kMaxTop) return "top_k must be between 0 and 32";
    return nullptr;
}
// Parts of a row: as many CTAs as the device holds at once, each with two
// vectors or more for every thread.  The quotient is rounded down, so a row count
// just above a divisor of the device's places leaves some of them empty, and one
// just above all of them starts a second wave.  128256 bf16 logits with 8
// alternatives: 394 rows (3 parts) 34.6 us, 395 (2) 36.9; 592 (2) 45.9, 593 (1)
// 48.5; 1184 68.3, 1185 (second wave) 84.6.
int logprobs_parts(int rows, int n, int dtype, int sms) {
    const long long vec = 16 / (long long)dtype_bytes(dtype);
    const long long most = std::min<long long>(lp::kMaxParts, n / (2 * vec * lp::kThreads));
    return int(std::max(1LL, std::min(most, (long long)lp::kCtas * sms / std::max(1, rows))));
}
struct LogprobsWs {
    size_t tickets, sums, keys, total;
};
// Rows are split while there are at most kCtas / 2 sms of them; the tickets' place
// does not depend on the call, so one workspace serves calls of other shapes.
LogprobsWs logprobs_ws(int rows, int parts, int top_k, int sms) {
    LogprobsWs w = {};
    if (parts > 1 && rows > 0) {
        const size_t cells = size_t(rows) * parts;
        w.tickets = round256(size_t(sms) * lp::kCtas / 2 * sizeof(unsigned));
        w.sums = round256(cells * sizeof(float4));
        w.keys = round256(cells * top_k * sizeof(unsigned long long));
        w.total = w.tickets + w.sums + w.keys;
    }
    return w;
}

}  // namespace
}  // namespace p100b

using namespace p100b;

extern "C" {

p100_status p100_paged_append(const p100_paged_desc* desc, const void* qkv, int qkv_type, long long qkv_stride,
                              const float* q_norm, const float* k_norm, float eps, const float* rope_cs, int max_pos,
                              int rope_half, const int* block_table, const int* q_start, const int* kv_len, void* q,
                              void* k_pages, void* v_pages, p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    paged::AppendParams prm = {};
    if (const char* why = paged_reason(*desc, prm.d)) return set_error(P100_ERR_INVALID, "%s", why);
    if (qkv_type != P100_F32 && qkv_type != P100_F16 && qkv_type != P100_BF16)
        return set_error(P100_ERR_INVALID, "unknown qkv type %d", qkv_type);
    const long long heads = (long long)desc->n_head_q + 2LL * desc->n_head_kv, width = heads * desc->head_dim;
    if (qkv_stride == 0) qkv_stride = width;
    if (qkv_stride < width) return set_error(P100_ERR_INVALID, "qkv_stride must be at least a fused row");
    if (qkv_stride * (qkv_type == P100_F32 ? 4 : 2) % 16)
        return set_error(P100_ERR_INVALID, "qkv rows must be 16-byte aligned");
    if ((q_norm || k_norm) && !(std::isfinite(eps) && eps >= 0.0f))
        return set_error(P100_ERR_INVALID, "eps must be finite and non-negative");
    if (rope_cs && max_pos <= 0) return set_error(P100_ERR_INVALID, "max_pos must be positive");
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (desc->n_tokens == 0 || desc->n_seq == 0) return P100_OK;
    if (!qkv || !block_table || !q_start || !kv_len || !q || !k_pages || !v_pages)
        return set_error(P100_ERR_INVALID, "null buffer");
    if (!aligned(qkv, 16) || !aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
        return set_error(P100_ERR_INVALID, "qkv, q and the pages must be 16-byte aligned");
    if (!aligned(rope_cs, 8)) return set_error(P100_ERR_INVALID, "rope_cs must be 8-byte aligned");
    prm.d.block_table = block_table;
    prm.d.q_start = q_start;
    prm.d.kv_len = kv_len;
    prm.qkv = qkv;
    prm.qkv_stride = qkv_stride;
    prm.q_norm = q_norm;
    prm.k_norm = k_norm;
    prm.eps = eps;
    prm.rope = reinterpret_cast<const float2*>(rope_cs);
    prm.max_pos = max_pos;
    prm.half = rope_half != 0;
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
    const long long blocks = ((long long)desc->n_tokens * prm.warps + paged::kAppendThreads / 32 - 1) / (paged::kAppendThreads / 32);
    if (blocks > INT_MAX) return set_error(P100_ERR_INVALID, "too many heads and tokens for one call");
    switch (qkv_type) {
        case P100_F32: return launch_append_to<float>(prm, desc->dtype, desc->head_dim, unsigned(blocks), stream);
        case P100_F16: return launch_append_to<__half>(prm, desc->dtype, desc->head_dim, unsigned(blocks), stream);
        default: return launch_append_to<__nv_bfloat16>(prm, desc->dtype, desc->head_dim, unsigned(blocks), stream);
    }
}

size_t p100_fa_paged_workspace_size(const p100_paged_desc* desc) {
    clear_error();
    paged::Desc d = {};
    int sms = 0;
    if (!desc) {
        set_error(P100_ERR_INVALID, "null descriptor");
        return 0;
    }
    if (const char* why = paged_reason(*desc, d)) {
        set_error(P100_ERR_INVALID, "%s", why);
        return 0;
    }
    if (require_sm100(nullptr, &sms)) return 0;
    return fa_paged_ws(*desc, sms).total;
}

p100_status p100_fa_paged_workspace_init(void* ws, size_t ws_bytes, p100_stream_t stream) {
    clear_error();
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (!ws || !ws_bytes) return P100_OK;
    return cuda_status(cudaMemsetAsync(ws, 0, std::min(ws_bytes, fa_paged_ticket_bytes(sms)), stream),
                       "cudaMemsetAsync(workspace)");
}

p100_status p100_fa_paged(const p100_paged_desc* desc, const void* q, const void* k_pages, const void* v_pages,
                          const int* block_table, const int* q_start, const int* kv_len, void* o, float* lse, void* ws,
                          size_t ws_bytes, p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    fap::Params prm = {};
    if (const char* why = paged_reason(*desc, prm.d)) return set_error(P100_ERR_INVALID, "%s", why);
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (desc->n_tokens == 0 || desc->n_seq == 0) return P100_OK;
    if (!q || !k_pages || !v_pages || !block_table || !q_start || !kv_len || !o)
        return set_error(P100_ERR_INVALID, "null buffer");
    if (o == q) return set_error(P100_ERR_INVALID, "o must not be q");
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
        return set_error(P100_ERR_INVALID, "q, o and the pages must be 16-byte aligned");
    const bool on_tc = fa_paged_on_tc(prm.d);
    if (on_tc ? fa_paged_too_long(prm.d, fatc::kRows, fatc::kKeys, fatc::kOver)
              : fa_paged_too_long(prm.d, fap::kRows, fap::kKeys, fap::kOver))
        return set_error(P100_ERR_INVALID, "max_q x max_pages x page_size is too long for one call");
    const FaPagedWs w = fa_paged_ws(*desc, sms);
    if (ws_bytes < w.total || !ws)
        return set_error(P100_ERR_INVALID, "workspace of %zu bytes needed, %zu given", w.total, ws ? ws_bytes : size_t(0));
    if (!aligned(ws, 256)) return set_error(P100_ERR_INVALID, "workspace must be 256-byte aligned");
    prm.d.block_table = block_table;
    prm.d.q_start = q_start;
    prm.d.kv_len = kv_len;
    prm.q = q;
    prm.k = k_pages;
    prm.v = v_pages;
    prm.o = o;
    prm.o_f32 = desc->o_fp32 != 0;
    prm.lse = lse;
    uint8_t* at = static_cast<uint8_t*>(ws);
    prm.tickets = reinterpret_cast<unsigned*>(at);
    prm.ws_o = reinterpret_cast<float*>(at + w.tickets);
    prm.ws_ml = reinterpret_cast<float*>(at + w.tickets + w.o);
    prm.scale = desc->scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(desc->head_dim)) : desc->scale;
    prm.softcap = desc->softcap;
    if (on_tc) {
        fatc::Params t = {};
        t.d = prm.d;
        t.q = prm.q;
        t.o = prm.o;
        t.o_f32 = prm.o_f32;
        t.lse = prm.lse;
        t.ws_o = prm.ws_o;
        t.ws_ml = prm.ws_ml;
        t.tickets = prm.tickets;
        t.scale = prm.scale;
        t.softcap = prm.softcap;
        t.k = k_pages;
        t.v = v_pages;
        // boxes of whole rows where 16 or more divide a page (a 4096-token
        // prompt over pages of 16: 170 us, gathered 207), else gathered rows
        // (pages of 24: 199 us, by boxes of 8 214)
        t.box = std::min(fatc::kKeys, prm.d.page_size & -prm.d.page_size);
        CUtensorMap tmk = {}, tmv = {};
        if (t.box < 16) {
            t.box = 0;
        } else {
            if (p100_status st = page_map(&tmk, k_pages, *desc, prm.d, t.box)) return st;
            if (p100_status st = page_map(&tmv, v_pages, *desc, prm.d, t.box)) return st;
        }
        return desc->dtype == P100_F16 ? launch_fa_paged_tc_d<__half>(t, desc->head_dim, tmk, tmv, sms, stream)
                                       : launch_fa_paged_tc_d<__nv_bfloat16>(t, desc->head_dim, tmk, tmv, sms, stream);
    }
    return desc->dtype == P100_F16 ? launch_fa_paged_mma_d<__half>(prm, desc->head_dim, sms, stream)
                                   : launch_fa_paged_mma_d<__nv_bfloat16>(prm, desc->head_dim, sms, stream);
}

size_t p100_logprobs_workspace_size(int rows, int n, int dtype, int top_k) {
    clear_error();
    int sms = 0;
    if (const char* why = logprobs_reason(rows, n, dtype, top_k)) {
        set_error(P100_ERR_INVALID, "%s", why);
        return 0;
    }
    if (require_sm100(nullptr, &sms)) return 0;
    return logprobs_ws(rows, logprobs_parts(rows, n, dtype, sms), top_k, sms).total;
}

p100_status p100_logprobs_workspace_init(void* ws, size_t ws_bytes, p100_stream_t stream) {
    clear_error();
    if (p100_status st = require_sm100(nullptr, nullptr)) return st;
    if (!ws || !ws_bytes) return P100_OK;
    return cuda_status(cudaMemsetAsync(ws, 0, ws_bytes, stream), "cudaMemsetAsync(workspace)");
}

p100_status p100_logprobs(const void* logits, int dtype, int n, int rows, long long row_stride, const int* token,
                          int top_k, float* logprob, float* entropy, int* rank, int* top_index, float* top_logprob,
                          void* ws, size_t ws_bytes, p100_stream_t stream) {
    clear_error();
    if (const char* why = logprobs_reason(rows, n, dtype, top_k)) return set_error(P100_ERR_INVALID, "%s", why);
    if (row_stride == 0) row_stride = n;
    if (row_stride < n) return set_error(P100_ERR_INVALID, "row_stride must be at least n");
    if ((logprob || rank) && !token) return set_error(P100_ERR_INVALID, "logprob and rank need tokens");
    if (top_k > 0 && (!top_index || !top_logprob))
        return set_error(P100_ERR_INVALID, "top_k needs top_index and top_logprob");
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (rows == 0) return P100_OK;
    if (!logits) return set_error(P100_ERR_INVALID, "null buffer");
    if (!aligned(logits, dtype_bytes(dtype))) return set_error(P100_ERR_INVALID, "logits must be aligned to their type");
    lp::Params prm = {};
    prm.x = logits;
    prm.stride = row_stride;
    prm.n = n;
    prm.rows = rows;
    prm.parts = logprobs_parts(rows, n, dtype, sms);
    const int vec = int(16 / dtype_bytes(dtype));
    prm.part_len = int(((long long)n + (long long)prm.parts * vec - 1) / ((long long)prm.parts * vec)) * vec;
    const LogprobsWs w = logprobs_ws(rows, prm.parts, top_k, sms);
    if (w.total > ws_bytes || (w.total && !ws))
        return set_error(P100_ERR_INVALID, "workspace of %zu bytes needed, %zu given", w.total, ws ? ws_bytes : size_t(0));
    if (w.total && !aligned(ws, 256)) return set_error(P100_ERR_INVALID, "workspace must be 256-byte aligned");
    prm.top = top_k;
    prm.token = token;
    prm.logprob = logprob;
    prm.entropy = entropy;
    prm.rank = rank;
    prm.top_index = top_index;
    prm.top_logprob = top_logprob;
    if (w.total) {
        uint8_t* at = static_cast<uint8_t*>(ws);
        prm.tickets = reinterpret_cast<unsigned*>(at);
        prm.ws_sums = reinterpret_cast<float4*>(at + w.tickets);
        prm.ws_keys = reinterpret_cast<unsigned long long*>(at + w.tickets + w.sums);
    }
    if ((long long)rows * prm.parts > INT_MAX) return set_error(P100_ERR_INVALID, "too many rows for one call");
    const unsigned grid = unsigned(rows) * unsigned(prm.parts);
    switch (dtype) {
        case P100_F32: lp::logprobs_kernel<float><<<grid, lp::kThreads, 0, stream>>>(prm); break;
        case P100_F16: lp::logprobs_kernel<__half><<<grid, lp::kThreads, 0, stream>>>(prm); break;
        default: lp::logprobs_kernel<__nv_bfloat16><<<grid, lp::kThreads, 0, stream>>>(prm); break;
    }
    return cuda_status(cudaGetLastError(), "logprobs_kernel launch");
}

}  // extern "C"
