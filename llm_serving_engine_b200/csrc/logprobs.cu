// C-ABI entry point of the token log-probabilities (declared in include/lse_int8.h).
#include <cuda_runtime.h>

#include <climits>

#include "../../include/lse_int8.h"
#include "host.h"
#include "logprobs.cuh"

namespace lse {

cudaError_t logprobs_device_status(int *status, bool reset) {
    cudaError_t e = cudaMemcpyFromSymbol(status, g_device_status, sizeof(int));
    const int zero = LSE_OK;
    if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(g_device_status, &zero, sizeof(int));
    return e;
}

}  // namespace lse

using namespace lse;

extern "C" int lse_token_logprobs(const void *logits, int dtype, int64_t M, int64_t V, int64_t ld, const int64_t *tokens,
                                  int64_t top_k, float *logprob, float *entropy, float *top_logprobs, int64_t *top_ids,
                                  void *stream) {
    if (M < 0 || V <= 0 || top_k < 0 || top_k > V || ld < V) return LSE_ERR_INVALID_ARG;
    if (dtype != LSE_BF16 && dtype != LSE_F16 && dtype != LSE_F32) return LSE_ERR_UNSUPPORTED;
    if (M == 0) return LSE_OK;
    if (!logits || !entropy || (tokens && !logprob) || (top_k && (!top_logprobs || !top_ids))) return LSE_ERR_INVALID_ARG;
    if (M > INT32_MAX || V > INT32_MAX / 4 || top_k > LSE_LOGPROBS_MAX_TOP) return LSE_ERR_UNSUPPORTED;
    const uintptr_t el = dtype == LSE_F32 ? 4 : 2;
    auto off = [](const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
    if (off(logits, el) || off(tokens, 8) || off(logprob, 4) || off(entropy, 4) || off(top_logprobs, 4) || off(top_ids, 8))
        return LSE_ERR_ALIGNMENT;
    int dev = 0;
    if (int rc = host::current_device(&dev)) return rc;
    logprobs::Params p{};
    p.x = logits;
    p.ld = ld;
    p.tokens = tokens;
    p.logprob = logprob;
    p.entropy = entropy;
    p.top_logprob = top_logprobs;
    p.top_id = top_ids;
    p.M = static_cast<int>(M);
    p.V = static_cast<int>(V);
    p.k = static_cast<int>(top_k);
    // CTAs of a row: as many as are resident at once (3 an SM), as long as each of a CTA's warps has a group
    // (rows of 128256: one row with 5 alternatives 9.6 us, 17.5 with one CTA; 64 with 20 18.4 against 36.9)
    const int step = 128 * static_cast<int>(16 / el);  // logits of one warp's loads
    p.group = step;
    p.cluster = 1;
    // Too few groups (512 logits each) for so many alternatives: 16 bytes are one, in a single CTA (64 bf16 rows
    // of 32000 with 128: 54 us against 2608 with groups of 512, all of whose logits would be candidates;
    // 8192 with 20: 9.0 against 89)
    const int64_t steps = (V + 16 + step - 1) / step;
    const bool scarce = 8 * top_k > 7 * ((V + 16) / 512) && steps * 128 <= logprobs::FINE_GROUPS;
    while (!scarce && p.cluster < logprobs::MAX_CLUSTER && 2 * M * p.cluster <= 3 * host::num_sms(dev) &&
           V > static_cast<int64_t>(p.cluster) * logprobs::WARPS * step)
        p.cluster *= 2;
    const int limit = (p.cluster > 1 ? 256 : logprobs::MAX_GROUPS) / 2;  // two maxima a group
    auto groups = [&] { return (V + 16 + static_cast<int64_t>(p.group) * p.cluster - 1) / (static_cast<int64_t>(p.group) * p.cluster); };
    while (groups() > limit) p.group *= 2;
    p.groups = static_cast<int>(groups());
    p.fine = p.cluster == 1 && p.group == step && p.groups * 128 <= (scarce ? logprobs::FINE_GROUPS : logprobs::MAX_GROUPS);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute pdl[1], attr[2];
    if (M * p.cluster > INT32_MAX) return LSE_ERR_UNSUPPORTED;
    host::launch_config(cfg, pdl, dim3(static_cast<unsigned>(M * p.cluster)), dim3(logprobs::THREADS), 0, static_cast<cudaStream_t>(stream));
    attr[0] = pdl[0];
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(p.cluster), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = p.cluster > 1 ? 2 : 1;
    const auto kernel = dtype == LSE_F32 ? logprobs::rows_kernel<float>
                        : dtype == LSE_F16 ? logprobs::rows_kernel<__half> : logprobs::rows_kernel<__nv_bfloat16>;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    return e == cudaSuccess ? LSE_OK : host::cuda_error(e, "token_logprobs launch");
}
