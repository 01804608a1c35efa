// The calls on embeddings, layer norms and token log probabilities on the HIP runtime of recorder.cpp: one line of stdin is one call, one line
// of stdout its result.
//   lookup n vocab d bf16                           status, then "kernel<arguments>:workgroups" each
//   embedding_bwd n vocab d bf16 accumulate ws      as lookup; ws = bytes of scratch
//   embedding_bwd_bytes n vocab d bf16              its scratch
//   norm rows d residual bias
//   norm_bwd rows d resid bias ws
//   norm_bwd_bytes rows d
//   logprobs rows vocab width top bf16 entropy ws
//   logprobs_bytes rows vocab top bf16
//   logprobs_bwd rows vocab width bf16 entropy
#define main recorder_main
#include "recorder.cpp"
#undef main

int main() {
    alignas(16) static char p[16];               // stands for every tensor: nothing reads them
    float* f = reinterpret_cast<float*>(p);
    int32_t* i = reinterpret_cast<int32_t*>(p);
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        in >> what;
        uint64_t n[8] = {};
        for (uint64_t& v : n) in >> v;
        auto type = [&](int at) { return n[at] ? TYR_HIP_BF16 : TYR_HIP_F32; };
        auto given = [&](int at) { return n[at] ? p : nullptr; };
        launched.clear();
        if (what == "lookup")
            printf("%d", tyr_hip_embedding(p, TYR_HIP_I64, p, p, n[0], n[1], n[2], 1.0f, type(3), nullptr));
        else if (what == "embedding_bwd")
            printf("%d", tyr_hip_embedding_bwd(p, p, TYR_HIP_I32, p, n[0], n[1], n[2], 1.0f, (int)n[4], type(3), given(5), n[5], nullptr));
        else if (what == "embedding_bwd_bytes")
            printf("%zu", tyr_hip_embedding_bwd_workspace_bytes(n[0], n[1], n[2], type(3)));
        else if (what == "norm")
            printf("%d", tyr_hip_layernorm_residual(p, given(2), p, given(3), p, given(2), n[0], n[1], 1e-5f, nullptr));
        else if (what == "norm_bwd")
            printf("%d", tyr_hip_layernorm_residual_bwd(p, given(2), p, p, p, p, given(3), n[0], n[1], 1e-5f, given(4), n[4], nullptr));
        else if (what == "norm_bwd_bytes")
            printf("%zu", tyr_hip_layernorm_residual_bwd_workspace_bytes(n[0], n[1]));
        else if (what == "logprobs")
            printf("%d", tyr_hip_token_logprobs(p, p, TYR_HIP_I64, f, f, n[5] ? f : nullptr, f, i, n[0], n[1], n[2], n[3], type(4), given(6), n[6], nullptr));
        else if (what == "logprobs_bytes")
            printf("%zu", tyr_hip_token_logprobs_workspace_bytes(n[0], n[1], n[2], type(3)));
        else if (what == "logprobs_bwd")
            printf("%d", tyr_hip_token_logprobs_bwd(p, p, TYR_HIP_I32, f, n[4] ? f : nullptr, f, n[4] ? f : nullptr, nullptr, p, n[0], n[1], n[2], type(3),
                                                    nullptr));
        printf("%s\n", launched.c_str());
        fflush(stdout);
    }
}
