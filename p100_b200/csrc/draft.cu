// draft.cu — the extern "C" entry points of include/p100/b200.h for steps of
// decoding with drafted tokens over a paged cache: the plan, the trees' masks,
// the append with computed rotations, the attention of trees and the move of
// accepted rows.  A translation unit of its own, with its own g_device_error
// word, which p100_device_error reads through draft_device_error.
#include "fa_tree.cuh"
#include "paged_host.cuh"
#include "paged_plan.cuh"
#include "rope.cuh"

namespace p100b {

p100_status draft_device_error(int clear, int* value) {
    if (p100_status st = cuda_status(cudaMemcpyFromSymbol(value, g_device_error, sizeof *value), "read device flag"))
        return st;
    if (clear && *value) {
        const int zero = 0;
        return cuda_status(cudaMemcpyToSymbol(g_device_error, &zero, sizeof zero), "clear device flag");
    }
    return P100_OK;
}

namespace {

// ------------------------------------------------------------ plan
// One CTA of 256 threads for the smallest steps, of 1024 up to kPlanOne rows,
// else a cluster of eight.
constexpr int kPlanOne = 4096;

// ------------------------------------------------------------ rotation
const char* scaling_reason(int rope_dim, double theta, const p100_rope_scaling& s) {
    if (s.kind < P100_ROPE_NONE || s.kind > P100_ROPE_DIVISORS) return "unknown rope scaling";
    if (!(std::isfinite(s.mscale) && s.mscale >= 0.0)) return "mscale must be finite and non-negative";
    const bool has_factor = s.kind >= P100_ROPE_LINEAR && s.kind <= P100_ROPE_YARN;
    if (has_factor && !(std::isfinite(s.factor) && s.factor > 0.0)) return "factor must be positive and finite";
    if (s.kind == P100_ROPE_NTK && rope_dim < 4) return "NTK scaling needs rope_dim of at least 4";
    if (s.kind == P100_ROPE_BANDS || s.kind == P100_ROPE_YARN) {
        if (s.original <= 0) return "original must be positive";
        if (!(s.low > 0.0 && s.high > s.low && std::isfinite(s.high))) return "low and high must be positive, low below high";
        if (s.kind == P100_ROPE_YARN && theta <= 1.0) return "YARN scaling needs theta above 1";
    }
    if (s.kind == P100_ROPE_DIVISORS) {
        if (!s.divisors) return "divisors must be given";
        for (int i = 0; i < rope_dim / 2; ++i)
            if (!(std::isfinite(s.divisors[i]) && s.divisors[i] > 0.0)) return "divisors must be positive and finite";
    }
    return nullptr;
}

const char* rope_reason(const p100_rope* rope, const p100_paged_desc* desc) {
    if (!rope) return "rope must be given";
    if (rope->rope_dim < 2 || rope->rope_dim % 2) return "rope_dim must be even and at least 2";
    if (desc && rope->rope_dim > desc->head_dim) return "rope_dim must be at most head_dim";
    if (!std::isfinite(rope->mscale)) return "rope's mscale must be finite";
    return nullptr;
}

struct AppendRopeLaunch {
    const paged::AppendParams& prm;
    const paged::TurnParams turns;
    unsigned blocks;
    cudaStream_t stream;
    template <typename S, typename T, int D>
    p100_status operator()() const {
        paged::append_rope_kernel<S, T, D><<<blocks, paged::kRopeThreads, 0, stream>>>(prm, turns);
        return cuda_status(cudaGetLastError(), "append_rope_kernel launch");
    }
};

// Whether n ints at a and m at b share one.
bool overlap(const int* a, size_t n, const int* b, size_t m) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + m * sizeof(int) && y < x + n * sizeof(int);
}

// ------------------------------------------------------------ trees
const char* words_reason(int mask_words) {
    return mask_words < 1 || mask_words > P100_TREE_MAX_WORDS ? "mask_words must be between 1 and 32" : nullptr;
}

// Which kernel takes a call of so many rows a kv head (max_q x group).  Up to 16 both
// carry the probabilities in two parts, so the choice is one of time alone.
//   over 16        tensor cores (tcgen05), probabilities rounded once
//   9 to 16, D 128 tensor cores where the row tiles are fewer than the SMs (one
//                  sequence of 4096, 32 / 8 heads, 4 tokens: 17.7 us, on mma.sync
//                  23.7; 16 of them 44.4 and 45.2), else mma.sync (48 of 8192, 64 / 8
//                  heads, 2 tokens: 176 us, on tensor cores 182; 64 of 512, 32 / 32
//                  heads, 16 tokens: 116 and 130)
//   else           mma.sync (one token of the 48: 170 us and 200; 64 of 512, 32 / 32
//                  heads, 8 tokens: 83 and 123; heads of 64, 16 rows: 64 of 512 27
//                  and 44, 13 trees of 5 over 3001 21 and 33, one of 4096 16.4 and 16.4)
bool fa_tree_on_tc(const paged::Desc& d, int head_dim, int sms) {
    const long long rows = (long long)d.max_q * d.group;
    if (rows > fap::kRows) return true;
    return head_dim == 128 && rows > fap::kRows / 2 && (long long)d.n_seq * d.n_head_kv < sms;
}

template <typename T, int D, bool SPARE>
p100_status launch_fa_tree_mma(const fap::Params& prm, int sms, cudaStream_t stream) {
    static thread_local int configured[64] = {};
    auto kern = fap::fa_paged_kernel<T, D, SPARE, true>;
    constexpr size_t fixed = fap::smem_bytes<D>();
    if (p100_status st = allow_smem(kern, fixed + paged::Lengths::bytes(paged::kMaxSeq), configured,
                                    "cudaFuncSetAttribute(fa_tree)"))
        return st;
    kern<<<sms * kMmaCtas, fap::kThreads, fixed + paged::Lengths::bytes(prm.d.n_seq), stream>>>(prm);
    return cuda_status(cudaGetLastError(), "fa_paged_kernel (tree) launch");
}
template <typename T>
p100_status launch_fa_tree_mma_d(const fap::Params& prm, int head_dim, int sms, cudaStream_t s) {
    // 8 rows a kv head or fewer: the second parts of their probabilities take the other 8
    const bool spare = (long long)prm.d.max_q * prm.d.group <= fap::kRows / 2;
    if (head_dim == 64) return spare ? launch_fa_tree_mma<T, 64, true>(prm, sms, s) : launch_fa_tree_mma<T, 64, false>(prm, sms, s);
    return spare ? launch_fa_tree_mma<T, 128, true>(prm, sms, s) : launch_fa_tree_mma<T, 128, false>(prm, sms, s);
}

static_assert(sizeof(fatr::Cut) <= kCutBytes && fatr::kRows <= fatc::kRows, "workspace");
template <typename T, int D, bool CAP, bool TWO>
p100_status launch_fa_tree_tc(const fatr::Params& prm, const CUtensorMap& tmk, const CUtensorMap& tmv, int sms,
                              cudaStream_t stream) {
    static thread_local int configured[64] = {};
    auto kern = fatr::fa_tree_kernel<T, D, CAP, TWO>;
    constexpr size_t fixed = fatr::smem_bytes<D>();
    if (p100_status st = allow_smem(kern, fixed + paged::Lengths::bytes(paged::kMaxSeq), configured,
                                    "cudaFuncSetAttribute(fa_tree)"))
        return st;
    const size_t lengths = paged::Lengths::bytes(prm.d.n_seq);
    kern<<<sms, fatr::kThreads, fixed + lengths, stream>>>(prm, tmk, tmv);
    if (p100_status st = cuda_status(cudaGetLastError(), "fa_tree_kernel launch")) return st;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute dependent = {};
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(fatr::kJoinThreads);
    cfg.stream = stream;
    cfg.attrs = &dependent;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, fatr::fa_tree_join_kernel<T, D>, prm, sms), "fa_tree_join_kernel launch");
}
template <typename T>
p100_status launch_fa_tree_tc_d(const fatr::Params& prm, int head_dim, const CUtensorMap& tmk, const CUtensorMap& tmv,
                                int sms, cudaStream_t s) {
    const bool cap = prm.softcap != 0.0f;
    if (head_dim == 64)
        return cap ? launch_fa_tree_tc<T, 64, true, false>(prm, tmk, tmv, sms, s)
                   : launch_fa_tree_tc<T, 64, false, false>(prm, tmk, tmv, sms, s);
    if ((long long)prm.d.max_q * prm.d.group <= fap::kRows)
        return cap ? launch_fa_tree_tc<T, 128, true, true>(prm, tmk, tmv, sms, s)
                   : launch_fa_tree_tc<T, 128, false, true>(prm, tmk, tmv, sms, s);
    return cap ? launch_fa_tree_tc<T, 128, true, false>(prm, tmk, tmv, sms, s)
               : launch_fa_tree_tc<T, 128, false, false>(prm, tmk, tmv, sms, s);
}

}  // namespace
}  // namespace p100b

using namespace p100b;

extern "C" {

p100_status p100_paged_plan(const p100_paged_desc* desc, const int* length, const int* n_new, int* pool, int* held,
                            int* block_table, int* q_start, int* kv_len, long long* slot, int* position,
                            p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    paged::Desc d = {};
    if (const char* why = paged_reason(*desc, d)) return set_error(P100_ERR_INVALID, "%s", why);
    if (p100_status st = require_sm100(nullptr, nullptr)) return st;
    if (!pool || !q_start || (d.n_seq > 0 && (!length || !n_new || !held || !kv_len || (!block_table && d.max_pages > 0))))
        return set_error(P100_ERR_INVALID, "null buffer");
    paged::PlanParams p = {d.n_seq, d.n_tokens, d.page_size, d.n_pages, d.max_pages, length, n_new, pool,
                           held,    block_table, q_start,    kv_len,    slot,        position};
    const bool small = d.n_seq <= paged::kPlanSmall && d.n_tokens <= paged::kPlanSmall;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim = {8, 1, 1};
    cfg.gridDim = dim3(d.n_tokens > kPlanOne ? 8 : 1);
    cfg.blockDim = dim3(small ? paged::kPlanSmall : paged::kPlanThreads);
    cfg.stream = stream;
    cfg.attrs = &cluster;
    cfg.numAttrs = d.n_tokens > kPlanOne ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, paged::paged_plan_kernel, p), "paged_plan_kernel launch");
}

p100_status p100_paged_pool_init(const p100_paged_desc* desc, int* pool, int* held, int* block_table,
                                 p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    paged::Desc d = {};
    if (const char* why = paged_reason(*desc, d)) return set_error(P100_ERR_INVALID, "%s", why);
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (!pool || (d.n_seq > 0 && (!held || (!block_table && d.max_pages > 0))))
        return set_error(P100_ERR_INVALID, "null buffer");
    paged::paged_pool_kernel<<<sms, 512, 0, stream>>>(d.n_seq, d.n_pages, d.max_pages, pool, held, block_table);
    return cuda_status(cudaGetLastError(), "paged_pool_kernel launch");
}

p100_status p100_tree_mask(const int* parent, const int* q_start, const int* kv_len, int n_seq, int n_tokens,
                           int mask_words, unsigned* mask, int* position, p100_stream_t stream) {
    clear_error();
    if (n_seq < 0 || n_tokens < 0) return set_error(P100_ERR_INVALID, "counts must not be negative");
    if (n_seq > P100_PAGED_MAX_SEQ) return set_error(P100_ERR_INVALID, "n_seq exceeds P100_PAGED_MAX_SEQ");
    if (const char* why = words_reason(mask_words)) return set_error(P100_ERR_INVALID, "%s", why);
    if (p100_status st = require_sm100(nullptr, nullptr)) return st;
    if (n_seq == 0 || n_tokens == 0) return P100_OK;
    if (!parent || !q_start || !kv_len || !mask) return set_error(P100_ERR_INVALID, "null buffer");
    const paged::TreeParams p = {n_seq, n_tokens, mask_words, parent, q_start, kv_len, mask, position};
    paged::tree_mask_kernel<<<n_seq, paged::kTreeThreads, 0, stream>>>(p);
    return cuda_status(cudaGetLastError(), "tree_mask_kernel launch");
}

p100_status p100_rope_init(p100_rope* rope, int rope_dim, int half, double theta, const p100_rope_scaling* scaling) {
    clear_error();
    if (!rope) return set_error(P100_ERR_INVALID, "rope must be given");
    if (rope_dim < 2 || rope_dim % 2 || rope_dim > 128)
        return set_error(P100_ERR_INVALID, "rope_dim must be even, between 2 and 128");
    if (!(std::isfinite(theta) && theta > 0.0)) return set_error(P100_ERR_INVALID, "theta must be positive and finite");
    const p100_rope_scaling s = scaling ? *scaling : p100_rope_scaling{};
    if (const char* why = scaling_reason(rope_dim, theta, s)) return set_error(P100_ERR_INVALID, "%s", why);
    using real = long double;
    const real pi2 = 6.283185307179586476925286766559L, r = rope_dim;
    real base = theta;
    if (s.kind == P100_ROPE_NTK) base *= std::pow(real(s.factor), r / (r - 2));
    real lo = 0, hi = 0;
    if (s.kind == P100_ROPE_YARN) {
        auto at = [&](double turns) { return r * std::log(s.original / (turns * pi2)) / (2 * std::log(real(theta))); };
        lo = std::max(std::floor(at(s.high)), real(0));
        hi = std::min(std::ceil(at(s.low)), r - 1);
        if (hi <= lo) hi = lo + 0.001L;
    }
    p100_rope out = {};
    out.rope_dim = rope_dim;
    out.half = half != 0;
    out.mscale = s.mscale != 0.0 ? float(s.mscale)
               : s.kind == P100_ROPE_YARN && s.factor > 1.0 ? float(0.1 * std::log(s.factor) + 1.0) : 1.0f;
    for (int i = 0; i < rope_dim / 2; ++i) {
        real f = std::pow(base, -2 * i / r);
        switch (s.kind) {
            case P100_ROPE_LINEAR: f /= s.factor; break;
            case P100_ROPE_BANDS: {
                const real w = std::min(std::max((s.original * f / pi2 - s.low) / (s.high - s.low), real(0)), real(1));
                f = w * f + (1 - w) * f / s.factor;
                break;
            }
            case P100_ROPE_YARN: {
                const real w = std::min(std::max((i - lo) / (hi - lo), real(0)), real(1));
                f = f / s.factor * w + f * (1 - w);
                break;
            }
            case P100_ROPE_DIVISORS: f /= s.divisors[i]; break;
            default: break;
        }
        const real turns = f / pi2;
        if (!(turns < 9007199254740992.0L)) return set_error(P100_ERR_INVALID, "frequency of pair %d is too high", i);
        // whole turns a token are none
        const real part = std::floor((turns - std::floor(turns)) * 18446744073709551616.0L + 0.5L);
        out.turns[i] = part >= 18446744073709551616.0L ? 0 : (unsigned long long)part;
    }
    *rope = out;
    return P100_OK;
}

p100_status p100_paged_append_rope(const p100_paged_desc* desc, const void* qkv, int qkv_type, long long qkv_stride,
                                   const float* q_norm, const float* k_norm, float eps, const p100_rope* rope,
                                   const int* position, const int* block_table, const int* q_start, const int* kv_len,
                                   void* q, void* k_pages, void* v_pages, p100_stream_t stream) {
    clear_error();
    paged::AppendParams prm = {};
    unsigned blocks = 0;
    if (p100_status st = append_params(desc, qkv, qkv_type, qkv_stride, q_norm, k_norm, eps, rope_reason(rope, desc),
                                       block_table, q_start, kv_len, q, k_pages, v_pages, paged::kRopeThreads, prm, blocks))
        return st;
    if (!blocks) return P100_OK;
    return append_typed(qkv_type, desc->dtype, desc->head_dim,
                        AppendRopeLaunch{prm, paged::TurnParams{*rope, position}, blocks, stream});
}

p100_status p100_fa_tree(const p100_paged_desc* desc, const void* q, const void* k_pages, const void* v_pages,
                         const unsigned* mask, int mask_words, const int* block_table, const int* q_start,
                         const int* kv_len, void* o, float* lse, void* ws, size_t ws_bytes, p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    fap::Params prm = {};
    if (const char* why = paged_reason(*desc, prm.d)) return set_error(P100_ERR_INVALID, "%s", why);
    if (const char* why = words_reason(mask_words)) return set_error(P100_ERR_INVALID, "%s", why);
    int sms = 0;
    if (p100_status st = require_sm100(nullptr, &sms)) return st;
    if (desc->n_tokens == 0 || desc->n_seq == 0) return P100_OK;
    if (!q || !k_pages || !v_pages || !mask || !block_table || !q_start || !kv_len || !o)
        return set_error(P100_ERR_INVALID, "null buffer");
    if (o == q) return set_error(P100_ERR_INVALID, "o must not be q");
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
        return set_error(P100_ERR_INVALID, "q, o and the pages must be 16-byte aligned");
    prm.d.causal = 0;
    prm.d.max_q = std::min(prm.d.max_q, 32 * mask_words);
    const bool on_tc = fa_tree_on_tc(prm.d, desc->head_dim, sms);
    if (sms > fatr::kJoinThreads) return set_error(P100_ERR_UNSUPPORTED, "more SMs than the joining kernel expects");
    if (on_tc ? fa_paged_too_long(prm.d, fatr::kRows, fatr::kKeys, fatr::kOver)
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
    prm.mask = mask;
    prm.words = mask_words;
    uint8_t* at = static_cast<uint8_t*>(ws);
    prm.tickets = reinterpret_cast<unsigned*>(at);
    prm.ws_o = reinterpret_cast<float*>(at + w.tickets);
    prm.ws_ml = reinterpret_cast<float*>(at + w.tickets + w.o);
    prm.scale = desc->scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(desc->head_dim)) : desc->scale;
    prm.softcap = desc->softcap;
    if (on_tc) {
        fatr::Params t = {};
        t.d = prm.d;
        t.q = prm.q;
        t.o = prm.o;
        t.o_f32 = prm.o_f32;
        t.lse = prm.lse;
        t.ws_o = prm.ws_o;
        t.ws_ml = prm.ws_ml;
        t.cuts = reinterpret_cast<fatr::Cut*>(at + w.tickets + w.o + w.ml);
        t.scale = prm.scale;
        t.softcap = prm.softcap;
        t.k = k_pages;
        t.v = v_pages;
        t.mask = mask;
        t.words = mask_words;
        // boxes of whole rows where 16 or more divide a page, else gathered rows (as p100_fa_paged)
        t.box = std::min(fatr::kKeys, prm.d.page_size & -prm.d.page_size);
        CUtensorMap tmk = {}, tmv = {};
        if (t.box < 16 || desc->n_pages == 0) {
            t.box = 0;
        } else {
            if (p100_status st = page_map(&tmk, k_pages, *desc, prm.d, t.box)) return st;
            if (p100_status st = page_map(&tmv, v_pages, *desc, prm.d, t.box)) return st;
        }
        return desc->dtype == P100_F16 ? launch_fa_tree_tc_d<__half>(t, desc->head_dim, tmk, tmv, sms, stream)
                                       : launch_fa_tree_tc_d<__nv_bfloat16>(t, desc->head_dim, tmk, tmv, sms, stream);
    }
    return desc->dtype == P100_F16 ? launch_fa_tree_mma_d<__half>(prm, desc->head_dim, sms, stream)
                                   : launch_fa_tree_mma_d<__nv_bfloat16>(prm, desc->head_dim, sms, stream);
}

p100_status p100_paged_keep(const p100_paged_desc* desc, void* k_pages, void* v_pages, const int* keep,
                            const int* keep_len, const int* block_table, const int* q_start, const int* kv_len,
                            int* length, p100_stream_t stream) {
    clear_error();
    if (!desc) return set_error(P100_ERR_INVALID, "null descriptor");
    paged::KeepParams p = {};
    if (const char* why = paged_reason(*desc, p.d)) return set_error(P100_ERR_INVALID, "%s", why);
    if (p100_status st = require_sm100(nullptr, nullptr)) return st;
    if (desc->n_seq == 0) return P100_OK;
    if (!k_pages || !v_pages || (!keep && desc->n_tokens > 0) || !keep_len || !block_table || !q_start || !kv_len)
        return set_error(P100_ERR_INVALID, "null buffer");
    if (!aligned(k_pages, 16) || !aligned(v_pages, 16))
        return set_error(P100_ERR_INVALID, "the pages must be 16-byte aligned");
    if (k_pages == v_pages) return set_error(P100_ERR_INVALID, "v_pages must not be k_pages");
    // a sequence's blocks read them while one of them writes its length
    const size_t seqs = desc->n_seq;
    if (length && (overlap(length, seqs, kv_len, seqs) || overlap(length, seqs, keep_len, seqs) ||
                   overlap(length, seqs, q_start, seqs + 1) || overlap(length, seqs, keep, desc->n_tokens) ||
                   overlap(length, seqs, block_table, seqs * desc->max_pages)))
        return set_error(P100_ERR_INVALID, "length must not overlap the other arrays");
    p.d.block_table = block_table;
    p.d.q_start = q_start;
    p.d.kv_len = kv_len;
    p.k = static_cast<uint4*>(k_pages);
    p.v = static_cast<uint4*>(v_pages);
    p.keep = keep;
    p.keep_len = keep_len;
    p.length = length;
    const int chunks = desc->head_dim / 8;
    const long long columns = 2LL * desc->n_head_kv * chunks;
    if (columns > INT_MAX - paged::kKeepThreads) return set_error(P100_ERR_INVALID, "too many heads for one call");
    const dim3 grid(unsigned((columns + paged::kKeepThreads - 1) / paged::kKeepThreads), unsigned(desc->n_seq));
    paged::paged_keep_kernel<<<grid, paged::kKeepThreads, 0, stream>>>(p, chunks);
    return cuda_status(cudaGetLastError(), "paged_keep_kernel launch");
}

}  // extern "C"
