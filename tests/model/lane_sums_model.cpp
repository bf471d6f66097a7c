// The sums of scatter_sum over the lanes of a warp, enumerated: every sum has one lane that stores it, and shares that launches
// add to one after another come out right in whatever order the lanes run.  Exit status 0: all holds.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>

#include "lane_sums.cuh"

static int failures = 0;
#define EXPECT(ok, ...) do { if (!(ok)) { std::printf(__VA_ARGS__); std::printf("\n"); ++failures; } } while (0)

// The backward scan's sums over channels: NL lanes share a channel's states, four a lane, Parts lanes share an output.
template <int NL>
void backward_scan() {
    constexpr int Parts = NL < 16 ? 16 / NL : 1, Each = Parts < 4 ? 4 / Parts : 1;
    struct Store { int lane; int word; };
    std::vector<Store> stores;
    std::map<int, int> writers;
    for (int lane = 0; lane < 32; ++lane) {
        const int tok = lane / (Parts * NL), quad = lane % NL, first = hdla::scatter_at<4, Parts>(lane, NL);
        if (!hdla::scatter_owner<4, Parts>(lane, NL)) continue;
        for (int i = 0; i < Each; ++i) {
            const int word = (tok * NL + quad) * 4 + first + i;
            stores.push_back({lane, word});
            ++writers[word];
        }
    }
    const int tokens = std::max(1, 32 / (Parts * NL));
    EXPECT((int)writers.size() == tokens * NL * 4, "NL=%d: %zu of %d words are stored", NL, writers.size(), tokens * NL * 4);
    for (const auto& w : writers) EXPECT(w.second == 1, "NL=%d: word %d has %d lanes that store it", NL, w.first, w.second);
    // launches after the first add: every lane loads, adds and stores, in any interleaving
    std::mt19937 rng(NL);
    for (int round = 0; round < 200; ++round) {
        std::map<int, int> memory;
        std::vector<int> loaded(stores.size());
        std::vector<std::pair<int, int>> steps;              // (store, 0: load, 1: write)
        for (int k = 0; k < (int)stores.size(); ++k) { steps.push_back({k, 0}); steps.push_back({k, 1}); }
        std::shuffle(steps.begin(), steps.end(), rng);
        std::vector<bool> has(stores.size(), false);
        for (auto& s : steps) {
            if (!has[s.first]) { loaded[s.first] = memory[stores[s.first].word]; has[s.first] = true; }
            else memory[stores[s.first].word] = loaded[s.first] + 1;
        }
        for (const auto& w : memory) EXPECT(w.second == 1, "NL=%d: word %d was added %d times", NL, w.first, w.second);
    }
}

// scatter_sum itself, lane by lane: what is held from scatter_at on is the sum over the lanes.
template <int N, int M>
void sums(int low) {
    std::vector<std::vector<long>> v(32, std::vector<long>(N)), at;
    for (int l = 0; l < 32; ++l)
        for (int i = 0; i < N; ++i) v[l][i] = (l + 1) * 1000003L + (i + 1) * 7919L * (l % 5 + 1);
    const auto in = v;
    int n = N;
    for (int m = 1; m < M; m <<= 1) {
        at = v;
        if (n > 1) n >>= 1;
        else {
            for (int l = 0; l < 32; ++l) v[l][0] = at[l][0] + at[l ^ (m * low)][0];
            continue;
        }
        for (int l = 0; l < 32; ++l) {
            const bool up = l & (m * low), up2 = (l ^ (m * low)) & (m * low);
            for (int i = 0; i < n; ++i) v[l][i] = (up ? at[l][i + n] : at[l][i]) + (up2 ? at[l ^ (m * low)][i] : at[l ^ (m * low)][i + n]);
        }
    }
    for (int l = 0; l < 32; ++l)
        for (int i = 0; i < std::max(1, N / M); ++i) {
            long want = 0;
            for (int k = 0; k < M; ++k) want += in[(l & ~((M - 1) * low)) | (k * low)][hdla::scatter_at<N, M>(l, low) + i];
            EXPECT(v[l][i] == want, "N=%d M=%d low=%d lane %d sum %d", N, M, low, l, i);
        }
}

int main() {
    backward_scan<2>();
    backward_scan<4>();
    backward_scan<8>();
    backward_scan<16>();
    backward_scan<32>();
    sums<4, 8>(2); sums<4, 4>(4); sums<4, 2>(8); sums<4, 1>(16);
    sums<2, 2>(1); sums<4, 4>(1); sums<4, 16>(1); sums<4, 32>(1);
    return failures ? 1 : 0;
}
