// How attention_bwd.hip deals its work, checked on the host for a range of plans: every tile of every block belongs to one
// piece, every part that the merge kernels add is written by the piece that they take it from and by no other, and parts
// exist where the merge kernels are launched. Compiled with the emulator's rewritten source.
#include "attention_bwd.cpp"

#include <cstdio>
#include <cstdlib>
#include <vector>

namespace mi {
namespace {

struct Case {
    uint32_t bhs, nb, NT;
    int keys, causal, f32;
};
uint64_t plans = 0, shared_plans = 0;

#define MUST(c)                                                                                                        \
    do {                                                                                                               \
        if (!(c)) {                                                                                                    \
            std::printf("%s: bhs %u nb %u NT %u keys %d causal %d f32 %d: wgs %u whole %u quo %u rem %u\n", #c, x.bhs, \
                        x.nb, x.NT, x.keys, x.causal, x.f32, d.wgs, d.whole, d.quo, d.rem);                            \
            std::exit(1);                                                                                              \
        }                                                                                                              \
    } while (0)

template <bool KEYS>
void check(const Case& x) {
    const bool causal = x.causal != 0;
    const Deal d = deal<KEYS>(x.bhs, x.nb * kB, x.NT * kTile, causal, x.f32 != 0);
    MUST(d.nb == x.nb && d.NT == x.NT && d.wgs > 0);
    const uint64_t blocks = static_cast<uint64_t>(x.bhs) * x.nb;
    struct Block {
        uint32_t done = 0, parts = 0;
        bool alone = false;
    };
    std::vector<Block> seen(blocks);
    std::vector<int64_t> slots(2ull * d.wgs, -1);  // which block's part a slot holds
    bool any = false;
    // whole blocks first: a share may go on where another workgroup's whole blocks end
    for (int shares = 0; shares < 2; ++shares)
        for (uint32_t w = 0; w < d.wgs; ++w) {
            Pieces<KEYS> pc(d, causal, w);
            for (uint32_t n = 0; pc.next(); ++n) {
                if ((n < d.whole) == (shares != 0)) continue;
                MUST(pc.bh < x.bhs && pc.blk < x.nb);
                const uint64_t id = static_cast<uint64_t>(pc.bh) * x.nb + pc.blk;
                Block& b = seen[id];
                const uint32_t tiles = before<KEYS>(pc.blk + 1, d.NT, causal) - before<KEYS>(pc.blk, d.NT, causal);
                MUST(tiles >= 1 && tiles <= d.NT);
                MUST(pc.t0 == b.done && pc.t1 > pc.t0);
                if (shares == 0) {
                    MUST(pc.whole && pc.t1 == d.NT);
                    b.done = tiles;
                } else {
                    MUST(pc.t1 <= tiles);
                    MUST(pc.whole == (pc.t0 == 0 && pc.t1 == tiles));
                    b.done = pc.t1;
                }
                if (pc.whole) {
                    b.alone = true;
                    continue;
                }
                any = true;
                const uint64_t slot = 2ull * w + (pc.first ? 0 : 1);
                MUST(slots[slot] == -1);
                slots[slot] = static_cast<int64_t>(id);
                ++b.parts;
            }
        }
    for (uint64_t id = 0; id < blocks; ++id) {
        const uint32_t bh = static_cast<uint32_t>(id / x.nb), blk = static_cast<uint32_t>(id % x.nb);
        const Block& b = seen[id];
        MUST(b.done == before<KEYS>(blk + 1, d.NT, causal) - before<KEYS>(blk, d.NT, causal));
        const Parts<KEYS> ps(d, causal, bh, blk);
        MUST((ps.w0 == ps.w1) == b.alone);
        if (b.alone) continue;
        MUST(ps.w0 < ps.w1 && ps.w1 < d.wgs && b.parts == ps.w1 - ps.w0 + 1);
        for (uint32_t w = ps.w0; w <= ps.w1; ++w) MUST(slots[ps.slot(d, w)] == static_cast<int64_t>(id));
    }
    // no merge kernel and no memory for parts where every block is whole; causal plans of whole blocks may launch one in vain
    MUST(!any || !all_whole(d, x.bhs));
    ++plans;
    shared_plans += any;
}

void every(Case x) {
    for (x.causal = 0; x.causal < 2; ++x.causal)
        for (x.f32 = 0; x.f32 < 2; ++x.f32) {
            x.keys = 0;
            check<false>(x);
            x.keys = 1;
            check<true>(x);
        }
}

}  // namespace
}  // namespace mi

int main() {
    using namespace mi;
    const uint32_t few[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 11, 12, 15, 16, 20, 24, 31, 32, 33, 40, 63, 64, 65, 77};
    for (uint32_t bhs : few)
        for (uint32_t nb = 1; nb <= 40; nb += nb < 12 ? 1 : 3)
            for (uint32_t NT = 1; NT <= 80; NT += NT < 24 ? 1 : 7) every({bhs, nb, NT, 0, 0, 0});
    const uint32_t many[] = {127, 128, 129, 154, 200, 255, 256, 257, 340, 341, 342, 400, 511, 512, 513, 541, 600, 767, 768, 769, 900, 1000, 1023, 1024, 1025};
    for (uint32_t bhs : many)
        for (uint32_t nb = 1; nb <= 6; ++nb)
            for (uint32_t NT = 1; NT <= 12; ++NT) every({bhs, nb, NT, 0, 0, 0});
    // long rows, more workgroups than 16 bits count, more tiles than 31 bits do
    for (uint32_t NT : {127u, 128u, 1000u, 4097u, 20011u})
        for (uint32_t nb : {1u, 3u, 64u, 500u}) every({1, nb, NT, 0, 0, 0}), every({20, nb, NT, 0, 0, 0});
    for (uint32_t bhs : {65535u, 65536u, 70001u, 200003u}) every({bhs, 1, 3, 0, 0, 0}), every({bhs, 2, 5, 0, 0, 0}), every({bhs, 5, 9, 0, 0, 0});
    every({70001, 5, 20011, 0, 0, 0});
    std::printf("OK %llu plans, %llu with shared blocks\n", static_cast<unsigned long long>(plans), static_cast<unsigned long long>(shared_plans));
}
