// Host-side check of the rule by which the sampling kernel's exchanges take turns at their two sets of words
// (compiled by tests/test_sample_turns_cpu.py).  A block that is ahead writes the words of its next exchange before
// that exchange's barrier, while a block that is behind may still have to read those of the last one it passed the
// barrier of.  So in every order of exchanges within a block ('b') and within a cluster ('c'), what is written
// before the next barrier of a kind must not be what may still have to be read after the last.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>

#include "eii_sample.cuh"

// Both kinds on one turn: what the kernel must not do, to see that the check sees it.
struct OneTurn {
    int turn = 0;
    int next_block() { return turn ^= 1; }
    int next_cluster() { return turn ^= 1; }
};

template <class Turns>
bool sound(const std::string& order) {
    Turns t;
    int block = -1, cluster = -1;  // the sets that slow threads, slow blocks may still read
    for (char op : order) {
        int& unread = op == 'b' ? block : cluster;
        const int set = op == 'b' ? t.next_block() : t.next_cluster();
        if (set == unread) return false;
        unread = set;
    }
    return true;
}

int main() {
    long bad = 0;
    std::mt19937 rng(5);
    // a row with a small top-k: maximum, two rounds and the distance, the logits within it, the list, how many weigh
    // more than any outside, the list's search in some steps, the draw
    for (int steps = 0; steps < 8; ++steps) {
        std::string row = "bc" "bb" "c" "bc" "bc" "bc";
        row += std::string(steps, 'b') + "bc";
        if (!sound<eii::SampleTurns>(row + row + row)) ++bad;
    }
    for (int i = 0; i < 100000; ++i) {
        std::string order;
        for (int n = rng() % 60; n > 0; --n) order += rng() % 3 ? 'b' : 'c';
        if (!sound<eii::SampleTurns>(order)) ++bad;
    }
    if (sound<OneTurn>("c" "b" "c")) ++bad;
    printf("unsound orders %ld\n", bad);
    return bad != 0;
}
