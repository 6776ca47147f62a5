// mfr_f8gemm: checks, and the choice of a tile (f8gemm_kernel.hpp).
#include "f8gemm_kernel.hpp"

namespace {

using mfr::f8gemm::Params;

// The descriptor's checks (of shapes, layouts and pointers: no device is needed).
Params checked(const mfr_f8gemm_desc* desc) {
    using mfr::require;
    require(desc != nullptr, "f8gemm: null descriptor");
    const mfr_f8gemm_desc& d = *desc;
    require(d.m >= 0 && d.n >= 0 && d.k >= 0, "f8gemm: negative dimension");
    require(d.act >= MFR_ACT_NONE && d.act <= MFR_ACT_SILU, "f8gemm: unknown activation");
    const bool gated = d.up.values != nullptr;
    require(!gated || (d.c0 == nullptr && d.bias == nullptr),
            "f8gemm: the gated form takes no c0 and no bias");
    require(d.beta == 0.0f || d.c0 != nullptr, "f8gemm: beta requires c0");
    Params p{};
    p.m = d.m, p.n = d.n, p.k = d.k;
    p.a = mfr::f8::checked(d.a, d.m, d.k, 1, false, "f8gemm", "a");
    p.b = mfr::f8::checked(d.b, d.n, d.k, 128, false, "f8gemm", "b");
    if (gated) {
        p.up = mfr::f8::checked(d.up, d.n, d.k, 128, false, "f8gemm", "up");
    }
    if (d.out_f8.values != nullptr) {
        p.q = mfr::f8::checked(d.out_f8, d.m, d.n, 1, true, "f8gemm", "out_f8");
    }
    if (d.m == 0 || d.n == 0) {
        return p;
    }
    const bool add = d.c0 != nullptr && d.beta != 0.0f;
    require(d.c != nullptr || d.out_f8.values != nullptr,
            "f8gemm: neither c nor out_f8 is given");
    require(d.c == nullptr || d.c_rs >= d.n, "f8gemm: c has rows that overlap");
    require(!add || d.c0_rs >= d.n, "f8gemm: c0 has rows that overlap");
    require(!add || d.c0 != d.c || d.c0_rs == d.c_rs,
            "f8gemm: c0 in place of c needs its row stride");
    p.c = d.c, p.c_rs = d.c_rs;
    p.c0 = add ? d.c0 : nullptr, p.c0_rs = d.c0_rs;
    p.bias = d.bias;
    p.beta = d.beta, p.act = d.act;
    return p;
}

int64_t tiles(const Params& p, int64_t bm, int64_t bn) {
    return ((p.m + bm - 1) / bm) * ((p.n + bn - 1) / bn);
}

void run(const mfr_stream& s, const Params& p) {
    // The small tile where the large one leaves compute units without a tile.
    const bool large = tiles(p, 128, 128) >= s.compute_units;
    if (p.up.values != nullptr) {
        if (large) {
            mfr::f8gemm::launch_gated<128, 128, 2, 4>(s, p);
        } else {
            mfr::f8gemm::launch_gated<64, 128, 1, 4>(s, p);
        }
    } else if (large) {
        mfr::f8gemm::launch<128, 128, 2, 2>(s, p);
    } else {
        mfr::f8gemm::launch<64, 128, 1, 4>(s, p);
    }
}

} // namespace

extern "C" {

int mfr_f8gemm(mfr_stream_t stream, const mfr_f8gemm_desc* desc) {
    return mfr::guarded([&] {
        const Params p = checked(desc);
        auto& s = mfr::stream_of(stream);
        if (p.m == 0 || p.n == 0) {
            return;
        }
        run(s, p);
    });
}

} // extern "C"
