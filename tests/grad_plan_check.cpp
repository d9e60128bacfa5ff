// CPU check of what a backward pass of microscaled matrices does for its sizes (int4linear_b200/csrc/grad_plan.cuh): the form
// of each size that the GPU tests name, cuts that were measured to pay and not to, and for many sizes that parts are long
// enough, that every piece of the workspace has its room, and that nothing depends on which gradients are wanted.
// Prints "PLAN_OK <cases>".
#include <algorithm>
#include <cstdio>
#include <utility>
#include <vector>

#include "../int4linear_b200/csrc/grad_plan.cuh"

using namespace i4l;

static int cases = 0;

static bool workspace_ok(long long m, long long n, long long k, bool gated, bool want_dx, bool want_dw, int terms)
{
    const Plan p = plan(m, n, k, gated, want_dx, want_dw, terms);
    const long long matrices = gated ? 2 : 1;
    std::vector<std::pair<long long, long long>> pieces;  // begin, bytes
    if (gated || n % 8) for (int i = 0; i < matrices; ++i) pieces.push_back({p.d[i], m * p.ld * 2});
    if (p.fine) for (int i = 2; i < 4; ++i) pieces.push_back({p.d[i], m * p.ld * 2});
    if (!p.unpack && want_dx) for (int i = 0; i < matrices; ++i) pieces.push_back({p.w[i], n * k * 2});
    if (!p.unpack && want_dw) pieces.push_back({p.x, m * k * 2});
    if (want_dx && p.dx.parts > 1) pieces.push_back({p.partial[0], p.dx.parts * m * k * 4});
    if (want_dw && p.dw.parts > 1) for (int i = 0; i < matrices; ++i) pieces.push_back({p.partial[1 + i], p.dw.parts * n * k * 4});
    std::sort(pieces.begin(), pieces.end());
    long long end = 0;
    for (const auto& [at, bytes] : pieces) {
        if (at < end || at % 256) return false;
        end = at + bytes;
    }
    return p.ld >= n && p.ld % 8 == 0 && end <= p.bytes && p.bytes < end + 256;
}

static int check(long long m, long long n, long long k, bool gated, int terms)
{
    const Plan both = plan(m, n, k, gated, true, true, terms);
    if (terms && both.fine != (gated && terms == 2)) return 5;
    for (const Kind* kind : {&both.dx, &both.dw})
        if (kind->parts < 1 || kind->parts > kMaxParts || (kind->parts > 1 && kind->segments * kind->seg_steps / kind->parts < kMinPart)) return 1;
    for (int want = 1; want <= 3; ++want) {
        const bool dx = want & 1, dw = want & 2;
        const Plan p = plan(m, n, k, gated, dx, dw, terms);
        if (p.fine != both.fine || p.unpack != both.unpack || p.dx.parts != both.dx.parts || p.dw.parts != both.dw.parts) return 2;
        if (p.tiles_dx != (dx ? both.tiles_dx : 0) || p.tiles_dw != (dw ? both.tiles_dw : 0)) return 3;
        if (!workspace_ok(m, n, k, gated, dx, dw, terms)) return 4;
    }
    ++cases;
    return 0;
}

enum { kUnpack = 1, kExpand = 2, kFine = 4, kOneTerm = 8, kCutDx = 16, kWholeDx = 32, kCutDw = 64, kWholeDw = 128 };

static bool form(long long m, long long n, long long k, bool gated, int want)
{
    const Plan p = plan(m, n, k, gated, true, true);
    const int have = (p.unpack ? kUnpack : kExpand) | (p.fine ? kFine : kOneTerm) | (p.dx.parts > 1 ? kCutDx : kWholeDx) | (p.dw.parts > 1 ? kCutDw : kWholeDw);
    if ((have & want) == want) return true;
    std::printf("FAIL form of %s %lld x %lld x %lld: wanted %d, has %d (parts %d, %d)\n", gated ? "gated" : "linear", m, n, k, want, have, p.dx.parts, p.dw.parts);
    return false;
}

int main()
{
    bool ok = true;
    // Forms that the tests on the GPU go by.
    ok &= form(1030, 4096, 1056, false, kExpand) && form(1030, 4101, 1056, false, kExpand) && form(1030, 4100, 1056, false, kExpand);
    ok &= form(300, 4100, 1056, true, kUnpack | kOneTerm | kCutDx) && form(300, 4104, 1056, true, kUnpack | kOneTerm | kCutDx);
    ok &= form(512, 3000, 2080, true, kUnpack | kOneTerm) && form(1030, 4100, 1056, true, kExpand | kOneTerm);
    ok &= form(515, 2731, 1056, true, kExpand | kOneTerm | kCutDx) && form(70, 200, 96, false, kUnpack) && form(128, 128, 128, true, kUnpack | kFine);
    // Measured: cut against whole, both gradients and the input's alone, back to back.  To cut pays ...
    ok &= form(64, 8192, 4096, false, kCutDx);    // 47 us and 62, 27 and 60
    ok &= form(256, 8192, 4096, false, kCutDx);   // 57 and 63, 31 and 60
    ok &= form(25, 15680, 12224, true, kCutDx);   // 385 and 373, 168 and 208
    ok &= form(512, 8192, 4096, true, kCutDx);    // 166 and 157, 84 and 122
    ok &= form(4, 20000, 704, false, kCutDx);     // 30 and 134, 21 and 133
    ok &= form(5000, 40, 64, false, kCutDw);
    // ... and does not, where the partial sums' way through memory takes what the shorter rounds save.
    ok &= form(2048, 8192, 4096, true, kWholeDx);   // 505 and 462, 306 and 274
    ok &= form(2048, 14336, 4096, true, kWholeDx);  // 856 and 794, 504 and 475
    ok &= form(4096, 14336, 4096, true, kWholeDx);  // 1591 and 1569, 916 and 910; in short runs 1368 and 1352, 956 and 983
    ok &= form(4096, 4096, 8192, false, kWholeDx | kWholeDw);
    if (!ok) return 1;
    const long long rows[] = {1, 2, 16, 63, 64, 65, 300, 512, 513, 1021, 4096, 4097, 8192, 131072, 1 << 26};
    const long long ks[] = {32, 96, 256, 288, 1024, 1056, 4096, 8192, 14336, 1 << 26};
    for (long long m : rows)
        for (long long n : rows)
            for (long long k : ks)
                for (bool gated : {false, true})
                    for (int terms = 0; terms <= (gated ? 2 : 0); ++terms)
                        if (const int rc = check(m, n, k, gated, terms)) {
                            std::printf("FAIL %d: %s %lld x %lld x %lld, terms %d\n", rc, gated ? "gated" : "linear", m, n, k, terms);
                            return 1;
                        }
    std::printf("PLAN_OK %d\n", cases);
    return 0;
}
