// How attention over the 8-bit cache deals out its units, compiled from the kernels' own source (DEAL: a file with those parts of it) and run on
// the CPU: a thread a lane, shuffles and barriers by std::barrier.  Every CTA's run is compared with a plain walk along the line in 64 bits.
#include <algorithm>
#include <barrier>
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <memory>
#include <random>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __align__(n) alignas(n)
#define __shared__ static
using std::max;
using std::min;
struct __half { uint16_t bits; };
struct CUtensorMap { uint64_t words[16]; };

constexpr int CTA = 64;
struct Index { int x; };
thread_local Index threadIdx;
static std::barrier<> whole(CTA);
static std::unique_ptr<std::barrier<>> warps[CTA / 32];
static unsigned char slots[CTA][8];
static int any_of[CTA];

static void warp_meet() { warps[threadIdx.x / 32]->arrive_and_wait(); }
static void __syncthreads() { whole.arrive_and_wait(); }
static int __syncthreads_or(int v)
{
    any_of[threadIdx.x] = v;
    __syncthreads();
    int r = 0;
    for (int x : any_of) r |= x;
    __syncthreads();
    return r;
}
template <typename T> static T from_lane(T v, int lane)
{
    const int warp0 = threadIdx.x / 32 * 32;
    memcpy(slots[threadIdx.x], &v, sizeof(T));
    warp_meet();
    T r;
    memcpy(&r, slots[warp0 + lane], sizeof(T));
    warp_meet();
    return r;
}
template <typename T> static T __shfl_sync(unsigned, T v, int lane) { return from_lane(v, lane & 31); }
template <typename T> static T __shfl_up_sync(unsigned, T v, int o) { const int l = threadIdx.x & 31; return from_lane(v, l >= o ? l - o : l); }
template <typename T> static T __shfl_xor_sync(unsigned, T v, int o) { return from_lane(v, (threadIdx.x & 31) ^ o); }
static unsigned __ballot_sync(unsigned, bool v)
{
    unsigned r = 0;
    slots[threadIdx.x][0] = v;
    warp_meet();
    for (int i = 0; i < 32; ++i) r |= (unsigned)slots[threadIdx.x / 32 * 32 + i][0] << i;
    warp_meet();
    return r;
}
static int __ffs(unsigned x) { return __builtin_ffs((int)x); }

constexpr int BLOCK = 64;
#include DEAL

struct Run { int seq, head, t, u0, n; bool begins, ends; bool operator==(const Run&) const = default; };

static std::vector<std::vector<Run>> by_device_code(const AttnArgs& a, const Deal& d, int ctas)
{
    std::vector<std::vector<Run>> runs(ctas);
    auto lane = [&](int tid) {
        threadIdx.x = tid;
        for (int cta = 0; cta < ctas; ++cta) {
            const Start start = find_start<CTA>(a, d, cta, ctas);
            Walk w;
            bool more = w.begin(a, d, start);
            for (; more; more = w.next(a, d))
                if (tid == 37) runs[cta].push_back({w.seq, w.head, w.t, w.u0, w.n, w.begins, w.ends});
            __syncthreads();
        }
    };
    std::vector<std::thread> threads;
    for (int i = 0; i < CTA; ++i) threads.emplace_back(lane, i);
    for (auto& t : threads) t.join();
    return runs;
}

static std::vector<std::vector<Run>> plainly(const AttnArgs& a, const Deal& d, int ctas)
{
    struct Piece { int seq, head, t; long long lo, units, at; };
    std::vector<Piece> line;
    long long total = 0;
    for (int s = 0; s < a.c.seqs; ++s) {
        const long long pos = a.r.start[s], rows = std::min<long long>(a.r.row_start[s + 1] - a.r.row_start[s], a.c.capacity - pos), all = rows * d.group;
        if (pos < 0 || rows <= 0) continue;
        for (int h = 0; h < a.c.kv_heads; ++h)
            for (long long t = 0; t * d.tile < all; ++t) {
                const long long first = pos + t * d.tile / d.group, last = pos + (std::min(all, (t + 1) * d.tile) - 1) / d.group;
                const long long lo = std::max(0LL, first - d.window + 1) / BLOCK, units = last / BLOCK + 1 - lo;
                line.push_back({s, h, (int)t, lo, units, total + d.extra});
                total += d.extra + units;
            }
    }
    const long long share = std::max<long long>(d.least, (total + ctas - 1) / ctas);
    std::vector<std::vector<Run>> runs(ctas);
    for (int c = 0; c < ctas; ++c)
        for (const Piece& x : line) {
            const long long b = std::max(x.at, share * c), e = std::min(x.at + x.units, share * (c + 1));
            if (b < e) runs[c].push_back({x.seq, x.head, x.t, (int)(x.lo + b - x.at), (int)(e - b), b == x.at, e == x.at + x.units});
        }
    return runs;
}

static int bad = 0;
static void check(const char* name, std::vector<int> starts, std::vector<int> counts, int kv_heads, int capacity, const Deal& d, int ctas)
{
    std::vector<int> row_start = {0};
    for (int n : counts) row_start.push_back(row_start.back() + n);
    AttnArgs a = {};
    a.c.seqs = (int)starts.size();
    a.c.kv_heads = kv_heads;
    a.c.capacity = capacity;
    a.num_heads = kv_heads * d.group;
    a.window = d.window;
    a.r = {row_start.data(), starts.data(), row_start.back(), *std::max_element(counts.begin(), counts.end())};
    if (by_device_code(a, d, ctas) != plainly(a, d, ctas)) {
        printf("differs: %s\n", name);
        ++bad;
    }
}

int main()
{
    for (auto& w : warps) w = std::make_unique<std::barrier<>>(32);
    check("prompt", {0}, {4000}, 4, 4032, {7, 256, INT_MAX, 8, 4}, 148);
    check("portions", {6000, 9000, 3001}, {500, 401, 399}, 4, 9600, {4, 256, INT_MAX, 8, 4}, 60);
    check("single tokens", {2047, -1, 5999, 0}, {1, 1, 1, 1}, 8, 6016, {5, 8, INT_MAX, 4, 1}, 96);
    std::mt19937 rng(1);
    auto below = [&](int n) { return (int)(rng() % n); };
    for (int i = 0; i < 5; ++i) {
        const int seqs = 1 + below(9), groups[] = {1, 4, 5, 7, 16, 71};
        std::vector<int> starts, counts;
        for (int s = 0; s < seqs; ++s) { starts.push_back(below(5) ? below(3000) : -1); counts.push_back(below(300)); }
        check("drawn", starts, counts, 1 + below(4), 3392, {groups[below(6)], 256, below(2) ? INT_MAX : 1 + below(400), 8, 4}, 40);
    }
    // a head of more units than 32 bits count: a few hundred tiles of 2^24 units
    check("far portion", {(1 << 30) - 1024}, {1024}, 1, 1 << 30, {128, 256, INT_MAX, 8, 4}, 100);
    printf("%s\n", bad ? "failed" : "ok");
    return bad != 0;
}
