// C++ mirror of the operators between logits and an update: a step with known
// answers on one GPU, and what the calls refuse.
#include <cmath>
#include <cstdio>
#include <limits>

#include "kernix_b200.hpp"

static int failures = 0;
#define EXPECT(cond)                                                              \
    do {                                                                          \
        if (!(cond)) {                                                            \
            std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond);       \
            ++failures;                                                           \
        }                                                                         \
    } while (0)

template <typename F> static int status_of(F f) {
    try {
        f();
    } catch (const kernix::OpsError &e) {
        return e.status();
    }
    return KX_OK;
}

int main() {
    const double inf = std::numeric_limits<double>::infinity();
    kernix::CudaExecutor cuda;
    // rows [0, log 3], [log 2, masked] and, at temperature 2, twice those
    auto logits = cuda.upload<double>({0.0, 2 * std::log(3.0), 2 * std::log(2.0), -inf}, {2, 2});
    auto tokens = cuda.upload<int64_t>({1, 0}, {2});
    auto out = cuda.token_log_probs<double>(logits, tokens, 2.0, 2, true);
    auto lp = cuda.download(*out.log_probs), lse = cuda.download(*out.lse), ent = cuda.download(*out.entropy);
    auto top = cuda.download(*out.top_log_probs);
    auto ids = cuda.download(*out.top_tokens);
    const double h = std::log(4.0) - 0.75 * std::log(3.0);
    EXPECT(std::fabs(lp[0] - std::log(0.75)) < 1e-15 && lp[1] == 0.0);
    EXPECT(std::fabs(lse[0] - std::log(4.0)) < 1e-15 && std::fabs(lse[1] - std::log(2.0)) < 1e-15);
    EXPECT(std::fabs(ent[0] - h) < 1e-15 && ent[1] == 0.0);
    EXPECT(ids[0] == 1 && ids[1] == 0 && ids[2] == 0 && ids[3] == -1);
    EXPECT(std::fabs(top[1] - std::log(0.25)) < 1e-15 && top[3] == -inf);
    // d(lp)/dx = (1[token] - p) / 2
    auto ones = cuda.upload<double>({1.0, 1.0}, {2});
    auto grad = cuda.token_log_probs_backward<double>(logits, tokens, out, 2.0, &ones);
    auto g = cuda.download(grad);
    EXPECT(std::fabs(g[0] + 0.125) < 1e-15 && std::fabs(g[1] - 0.125) < 1e-15 && g[2] == 0.0 && g[3] == 0.0);
    // a 3-4-12 triple: norm 13, scaled in place to 6.5
    std::vector<kernix::DeviceTensor<float>> grads = {cuda.upload<float>({3.0f, 0.0f, 4.0f}, {3}),
                                                      cuda.upload<float>({0.0f, 12.0f}, {2, 1}).transpose()};
    EXPECT(cuda.download(cuda.grad_norm<float>(grads))[0] == 13.0f);
    EXPECT(cuda.download(cuda.clip_grad_norm<float>(grads, 6.5))[0] == 13.0f);
    EXPECT(cuda.download(grads[0])[2] == 2.0f && cuda.download(grads[1])[1] == 6.0f);
    EXPECT(cuda.download(cuda.clip_grad_norm<float>(grads, 7.0))[0] == 6.5f && cuda.download(grads[0])[0] == 1.5f);
    // refusals, in the library's words
    EXPECT(status_of([&] { cuda.token_log_probs<double>(logits, tokens, 0.0); }) == KX_E_PARAM);
    EXPECT(status_of([&] { cuda.token_log_probs<double>(logits, tokens, 1.0, 33); }) == KX_E_PARAM);
    EXPECT(status_of([&] { cuda.clip_grad_norm<float>(grads, -1.0); }) == KX_E_PARAM);
    EXPECT(status_of([&] { cuda.clip_grad_norm<float>({grads[0], grads[0]}, 1.0); }) == KX_E_ALIAS);
    if (failures) {
        std::fprintf(stderr, "%d failure(s)\n", failures);
        return 1;
    }
    std::printf("update_test ok\n");
    return 0;
}
