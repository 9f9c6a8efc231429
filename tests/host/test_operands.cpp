// operands.hpp against the bytes themselves: every pair of small operands with any pitches, widths, rows and offsets.
#include <cstdio>
#include <random>
#include <vector>

#include "../../backup_1_amd/csrc/operands.hpp"

using namespace decx_hip;

static bool bytes_meet(const Operand& a, const Operand& b, const unsigned char* base, size_t n) {
    std::vector<bool> in(n, false);
    if (!a.there() || !b.there()) return false;
    for (size_t i = 0; i < a.rows; ++i)
        for (size_t j = 0; j < a.width; ++j) in[(size_t)(static_cast<const unsigned char*>(a.p) - base) + i * a.pitch + j] = true;
    for (size_t i = 0; i < b.rows; ++i)
        for (size_t j = 0; j < b.width; ++j)
            if (in[(size_t)(static_cast<const unsigned char*>(b.p) - base) + i * b.pitch + j]) return true;
    return false;
}

int main() {
    static unsigned char base[256];
    int bad = 0, met = 0, nested = 0;
    std::mt19937 rng(7);
    for (int turn = 0; turn < 2000000; ++turn) {
        auto draw = [&](size_t pitch) {
            Operand o;
            o.rows = rng() % 6, o.width = rng() % (pitch + 1), o.pitch = pitch;
            o.p = rng() % 50 ? base + rng() % 100 : nullptr;
            return o;
        };
        const size_t pitch = 1 + rng() % 20;
        const Operand a = draw(pitch), b = draw(turn % 2 ? pitch : 1 + rng() % 20);
        const bool want = bytes_meet(a, b, base, sizeof(base)), got = operands_meet(a, b), turned = operands_meet(b, a);
        bad += want != got || want != turned;
        met += want;
        nested += a.there() && b.there() && !want && a.begin() < b.end() && b.begin() < a.end();
        if (want && operands_coincide(a, b)) bad += a.p != b.p;
    }
    const Operand x = operand(base, 3, 4, 8, 2), next = operand(base + 8, 3, 4, 8, 2), wide = operand(base, 3, 4, 9, 2);
    bad += !results_fit({{next, 0}}, {x});                                       // columns of one matrix
    bad += !results_fit({{x, 1}}, {x}) + results_fit({{x, 0}}, {x}) + results_fit({{x, 1}}, {x, x}) + !results_fit({{x, 3}}, {x, x});
    bad += results_fit({{wide, 1}}, {x});                                        // in place at another pitch
    bad += results_fit({{x, 1}, {x, 1}}, {x}) + !results_fit({{x, 0}, {next, 0}}, {});
    std::printf("%d pairs met, %d lay between each other: %d failure(s)\n", met, nested, bad);
    return bad || !met || !nested;
}
