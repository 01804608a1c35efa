// The calls on a cache in pages and of the RMS norm on the HIP runtime of recorder.cpp: one line of stdin is one call, one line of
// stdout its result.
//   decode B Hq Hkv D page width window sinks e4m3 ws   status, then "kernel<arguments>:workgroups" each; ws = bytes of scratch
//   decode_bytes B Hq Hkv D page width                  scratch of a decode
//   norm rows d residual e4m3 row_scale                 as decode; row_scale = an address
//   norm_bwd rows d resid ws
//   norm_bwd_bytes rows d
#define main recorder_main
#include "recorder.cpp"
#undef main

int main() {
    alignas(16) static char p[16];               // stands for every tensor: nothing reads them
    float* f = reinterpret_cast<float*>(p);
    const int32_t* i = reinterpret_cast<const int32_t*>(p);
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        in >> what;
        uint64_t n[10] = {};
        for (uint64_t& v : n) in >> v;
        launched.clear();
        if (what == "decode")
            printf("%d", tyr_hip_paged_decode(p, p, p, i, i, nullptr, nullptr, p, f, n[0], n[1], n[2], n[3], 1, n[4], n[5], n[6], n[7], (int)n[8],
                                              0.125f, n[9] ? p : nullptr, n[9], nullptr));
        else if (what == "decode_bytes")
            printf("%zu", tyr_hip_paged_decode_workspace_bytes(n[0], n[1], n[2], n[3], n[4], n[5]));
        else if (what == "norm")
            printf("%d", tyr_hip_rmsnorm_residual(p, n[2] ? p : nullptr, p, p, n[2] ? p : nullptr, reinterpret_cast<float*>(n[4]), n[0], n[1], 1e-6f,
                                                  n[3] ? TYR_HIP_OUT_E4M3 : TYR_HIP_OUT_BF16, nullptr));
        else if (what == "norm_bwd")
            printf("%d", tyr_hip_rmsnorm_residual_bwd(p, n[2] ? p : nullptr, p, p, p, p, n[0], n[1], 1e-6f, n[3] ? p : nullptr, n[3], nullptr));
        else if (what == "norm_bwd_bytes")
            printf("%zu", tyr_hip_rmsnorm_residual_bwd_workspace_bytes(n[0], n[1]));
        printf("%s\n", launched.c_str());
        fflush(stdout);
    }
}
