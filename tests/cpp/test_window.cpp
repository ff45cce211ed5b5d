// flash_attention_windowed_forward of include/brotensor/ops.h with a window, against its definition in
// double precision on the host; window 0 against the causal operator.
#include <cmath>
#include <cstdio>
#include <random>
#include <tuple>
#include <vector>

#include "brotensor/ops.h"

namespace bt = brotensor;

static std::vector<float> host(const bt::Tensor& t) {
    const auto raw = t.to_host_bytes();
    const auto* b = reinterpret_cast<const std::uint16_t*>(raw.data());
    std::vector<float> out(t.size());
    for (std::size_t i = 0; i < out.size(); ++i) out[i] = bt::bf16_bits_to_fp32(b[i]);
    return out;
}
static bt::Tensor random_rows(std::mt19937& rng, int rows, int cols, std::vector<float>& values) {
    std::normal_distribution<float> d;
    std::vector<std::uint16_t> bits(static_cast<std::size_t>(rows) * cols);
    values.resize(bits.size());
    for (std::size_t i = 0; i < bits.size(); ++i) {
        bits[i] = bt::fp32_to_bf16_bits(d(rng));
        values[i] = bt::bf16_bits_to_fp32(bits[i]);
    }
    return bt::Tensor::from_host_bf16(bits.data(), rows, cols);
}

int main() {
    std::mt19937 rng(7);
    const int nh = 2, hd = 64, D = nh * hd;
    int failures = 0;
    for (const auto& [lq, lk, window] : {std::tuple<int, int, int>{1, 90, 20}, {50, 170, 33}, {150, 150, 1}, {150, 200, 64}, {9, 40, 500}}) {
        std::vector<float> q, k, v;
        const bt::Tensor Q = random_rows(rng, lq, D, q), K = random_rows(rng, lk, D, k), V = random_rows(rng, lk, D, v);
        bt::Tensor O;
        bt::flash_attention_windowed_forward(Q, K, V, nullptr, nh, window, O);
        const std::vector<float> o = host(O);
        double worst = 0.0;
        for (int i = 0; i < lq; ++i) {
            for (int h = 0; h < nh; ++h) {
                const int pos = lk - lq + i, first = pos - window + 1 > 0 ? pos - window + 1 : 0;
                std::vector<double> p;
                double sum = 0.0;
                for (int j = first; j <= pos; ++j) {
                    double s = 0.0;
                    for (int c = 0; c < hd; ++c) s += static_cast<double>(q[i * D + h * hd + c]) * k[j * D + h * hd + c];
                    p.push_back(std::exp(s / 8.0));
                    sum += p.back();
                }
                for (int c = 0; c < hd; ++c) {
                    double ref = 0.0, mag = 0.0;
                    for (int j = first; j <= pos; ++j) {
                        ref += p[j - first] / sum * v[j * D + h * hd + c];
                        mag += p[j - first] / sum * std::fabs(v[j * D + h * hd + c]);
                    }
                    // output and weights rounded to BF16 (2^-8 each), FP32 scores below 3e-4
                    const double bound = std::fabs(ref) / 256 + (1.0 / 256 + 3e-4) * mag;
                    const double err = std::fabs(o[i * D + h * hd + c] - ref) / bound;
                    if (!(err <= worst)) worst = err;
                }
            }
        }
        std::printf("  %d queries, %d keys, window %d: %.3f of the bound\n", lq, lk, window, worst);
        if (!(worst <= 1.0)) ++failures;
        bt::Tensor A, B;
        bt::flash_attention_windowed_forward(Q, K, V, nullptr, nh, 0, A);
        bt::flash_attention_forward(Q, K, V, nullptr, nh, true, B);
        if (host(A) != host(B)) ++failures;
        try {
            bt::flash_attention_windowed_forward(Q, K, V, nullptr, nh, -1, A);
            ++failures;
        } catch (const std::runtime_error&) {
        }
    }
    if (failures == 0) std::printf("test_window: ok\n");
    return failures != 0;
}
