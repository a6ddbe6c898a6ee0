// The plans of the 8-bit products depend on the device that is passed and on nothing that another device's calls leave behind: two devices of different
// sizes, one without the pair kernel, planned by threads side by side.
#include <cstdio>
#include <cstring>
#include <thread>
#include <vector>

#include "../venom_b200/csrc/vnm_fp8.h"

using namespace vnm;

namespace {

struct Plans {
    Fp8Plan small, pair;
    float small_us, pair_us;
};
const int shapes[][3] = {{1, 8, 16}, {8, 1024, 1024}, {16, 36864, 12288}, {512, 4096, 4096}, {16384, 4096, 1024}, {2049, 515, 384}, {333, 1537, 776}};

Plans plans_of(const int *s, const Fp8Device &d)
{
    Plans p;
    std::memset(&p, 0, sizeof(p));
    p.small_us = fp8_small_config(s[0], s[1], (s[2] + 127) / 128, false, d, &p.small);
    p.pair_us = fp8_pair_config(s[0], s[1], s[2], false, true, false, d, &p.pair);
    return p;
}
bool same(const Fp8Plan &a, const Fp8Plan &b) { return a.bn == b.bn && a.split == b.split && a.grid == b.grid; }

}  // namespace

int main()
{
    const Fp8Device devices[] = {{148, 74}, {64, 32}, {148, 0}};
    bool good = true, differ = false;
    std::vector<Plans> alone[3];
    for (int d = 0; d < 3; d++)
        for (const auto &s : shapes) alone[d].push_back(plans_of(s, devices[d]));
    for (size_t i = 0; i < alone[0].size(); i++) {
        good = good && alone[2][i].pair_us < 0.0f && alone[0][i].pair.grid <= 148 && alone[1][i].pair.grid <= 64;
        differ = differ || alone[0][i].pair.grid != alone[1][i].pair.grid;
    }
    bool kept[3] = {true, true, true};
    std::vector<std::thread> threads;
    for (int d = 0; d < 3; d++)
        threads.emplace_back([&, d] {
            for (int round = 0; round < 2000; round++)
                for (size_t i = 0; i < alone[d].size(); i++) {
                    const Plans p = plans_of(shapes[i], devices[d]);
                    kept[d] = kept[d] && p.small_us == alone[d][i].small_us && p.pair_us == alone[d][i].pair_us && same(p.small, alone[d][i].small) && same(p.pair, alone[d][i].pair);
                }
        });
    for (auto &t : threads) t.join();
    if (!good || !differ || !kept[0] || !kept[1] || !kept[2]) return std::printf("plans differ\n"), 1;
    std::printf("plans ok\n");
    return 0;
}
