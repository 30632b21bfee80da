// GPU: the paged-cache operators through the C++ host side, as a server would call them: prompts of
// different lengths rotated and appended to 4-bit pages, attended as packed rows, read back, and one
// more token each attended over the pages.  Checked against float64 loops on the same seeded inputs:
// normwise 1e-2 for bf16 outputs, a 4-bit value by half a step of its group and the roundings of
// the group's f16 scale and offset.
#include <algorithm>
#include <numeric>

#include "backend.hpp"
#include "check.hpp"
#include "oracle.h"

using namespace puter::hip;
using check::normal;
using check::normwise;

namespace {

constexpr int64_t QH = 8, KV = 2, D = 128, G = 64, PS = 16;

Backend &be() {
    static Backend b;
    return b;
}

std::vector<uint8_t> encode(const std::vector<float> &x, DType dt) {
    std::vector<uint8_t> out((size_t)ByteCount(dt, (int64_t)x.size()));
    or_cast_from_f32(out.data(), x.data(), x.size(), static_cast<int>(dt));
    return out;
}

std::vector<float> decode(const std::vector<uint8_t> &bits, DType dt, size_t n) {
    std::vector<float> out(n);
    or_cast_to_f32(out.data(), bits.data(), n, static_cast<int>(dt));
    return out;
}

template <class T> Tensor upload(const std::vector<T> &host, std::vector<int64_t> shape, DType dt) {
    Tensor t = be().AllocateTensor(std::move(shape), dt);
    be().Upload(t.data, host.data(), host.size() * sizeof(T));
    return t;
}

std::vector<float> download_f32(const Tensor &t, DType dt) {
    std::vector<uint8_t> out((size_t)t.byteCount);
    be().Download(out.data(), t.data, out.size());
    return decode(out, dt, (size_t)t.Numel());
}

// rows of [heads * D] rotated at their positions, pairs D / 2 apart
std::vector<float> rotated(std::vector<float> x, int64_t heads, const std::vector<int32_t> &pos) {
    for (size_t r = 0; r < pos.size(); ++r)
        for (int64_t h = 0; h < heads; ++h)
            for (int64_t i = 0; i < D / 2; ++i) {
                float *p = &x[(r * heads + h) * D + i];
                const double a = pos[r] * std::pow(10000.0, -2.0 * i / D), c = std::cos(a), s = std::sin(a), u = p[0], v = p[D / 2];
                p[0] = (float)(u * c - v * s);
                p[D / 2] = (float)(u * s + v * c);
            }
    return x;
}

// one query row of QH heads over n rows of keys and values
std::vector<float> attend(const float *q, const float *k, const float *v, int64_t n) {
    std::vector<float> out((size_t)(QH * D), 0.0f);
    for (int64_t h = 0; h < QH; ++h) {
        const int64_t kvh = h / (QH / KV);
        std::vector<double> s((size_t)n);
        double top = -1e300, sum = 0.0;
        for (int64_t t = 0; t < n; ++t) {
            double dot = 0.0;
            for (int64_t d = 0; d < D; ++d) dot += (double)q[h * D + d] * k[(t * KV + kvh) * D + d];
            top = std::max(top, s[t] = dot / std::sqrt((double)D));
        }
        std::vector<double> o((size_t)D, 0.0);
        for (int64_t t = 0; t < n; ++t) {
            const double p = std::exp(s[t] - top);
            sum += p;
            for (int64_t d = 0; d < D; ++d) o[d] += p * v[(t * KV + kvh) * D + d];
        }
        for (int64_t d = 0; d < D; ++d) out[h * D + d] = (float)(o[d] / sum);
    }
    return out;
}

struct Cache {
    std::vector<int32_t> table;   // [sequence][pages]
    int64_t pages, per;
    Tensor k, v, kp, vp;
    Cache(int64_t batch, int64_t per_sequence) : table((size_t)(batch * per_sequence)), pages(batch * per_sequence), per(per_sequence) {
        std::iota(table.begin(), table.end(), 0);
        std::reverse(table.begin(), table.end());
        k = be().AllocateTensor({pages, PS, KV, D}, DType::Int4), v = be().AllocateTensor({pages, PS, KV, D}, DType::Int4);
        kp = be().AllocateTensor({pages, PS, KV, D / G, 2}, DType::Float16);
        vp = be().AllocateTensor({pages, PS, KV, D / G, 2}, DType::Float16);
    }
};

// fused rows [q | k | v] into the cache; the rotated queries
Tensor append(const Cache &c, const Tensor &qkv, int64_t rows, const std::vector<int32_t> &pos, const std::vector<int32_t> &ids,
              const std::vector<int32_t> &slots) {
    RoPEConfig cfg;
    cfg.Mode = RoPEModeHalf;
    Tensor q = be().AllocateTensor({rows, QH * D}, DType::BFloat16);
    Tensor dp = upload(pos, {rows}, DType::Int32), di = upload(ids, {rows}, DType::Int32), ds = upload(slots, {rows}, DType::Int32);
    const char *x = static_cast<const char *>(qkv.data);
    const int64_t stride = (QH + 2 * KV) * D;
    be().KVPageAppendRoPE(&cfg, x, x + QH * D * 2, x + (QH + KV) * D * 2, dp.data, di.data, ds.data, q.data, c.k.data, c.v.data, c.kp.data,
                          c.vp.data, rows, QH, KV, D, stride, stride, stride, c.pages, PS, G, DType::BFloat16, DType::Int4);
    be().CheckStatus();
    return q;
}

std::vector<float> gathered(const Cache &c, const Tensor &pool, const Tensor &par, int64_t b, int64_t rows) {
    Tensor t = upload(std::vector<int32_t>(c.table.begin() + b * c.per, c.table.begin() + (b + 1) * c.per), {c.per}, DType::Int32);
    Tensor out = be().AllocateTensor({rows, KV * D}, DType::Float32);
    be().KVPageGatherInt4(pool.data, par.data, t.data, out.data, c.pages, PS, KV, D, G, rows, DType::Float32);
    be().CheckStatus();
    return download_f32(out, DType::Float32);
}

void split(const std::vector<float> &x, int64_t rows, std::vector<float> &q, std::vector<float> &k, std::vector<float> &v) {
    const int64_t w = (QH + 2 * KV) * D;
    for (int64_t r = 0; r < rows; ++r) {
        q.insert(q.end(), &x[r * w], &x[r * w] + QH * D);
        k.insert(k.end(), &x[r * w + QH * D], &x[r * w] + (QH + KV) * D);
        v.insert(v.end(), &x[r * w + (QH + KV) * D], &x[r * w] + w);
    }
}

}  // namespace

CASE(prompts_then_a_token_over_4_bit_pages) {
    const std::vector<int32_t> lens = {37, 90, 1};
    const int64_t B = 3, per = 6, W = (QH + 2 * KV) * D;
    Cache c(B, per);
    std::vector<int32_t> pos, ids, slots, off = {0};
    for (int64_t b = 0; b < B; ++b) {
        for (int32_t t = 0; t < lens[b]; ++t) {
            pos.push_back(t);
            ids.push_back(c.table[b * per + t / PS]);
            slots.push_back(t % PS);
        }
        off.push_back(off.back() + lens[b]);
    }
    const int64_t rows = off.back();
    auto bits = encode(normal(701, rows * W), DType::BFloat16);
    std::vector<float> q, k, v;
    split(decode(bits, DType::BFloat16, rows * W), rows, q, k, v);
    Tensor x = upload(bits, {rows, W}, DType::BFloat16);
    Tensor dq = append(c, x, rows, pos, ids, slots);
    q = rotated(q, QH, pos), k = rotated(k, KV, pos);
    EXPECT(normwise(download_f32(dq, DType::BFloat16), q) <= 1e-2, "rotated queries");

    // the prompts among themselves, their own rows of K and V
    auto kb = encode(k, DType::BFloat16), vb = encode(v, DType::BFloat16);
    Tensor dk = upload(kb, {rows, KV * D}, DType::BFloat16), dv = upload(vb, {rows, KV * D}, DType::BFloat16);
    Tensor doff = upload(off, {B + 1}, DType::Int32), o = be().AllocateTensor({rows, QH * D}, DType::BFloat16);
    MultiHeadAttentionConfig cfg;
    cfg.NumHeads = QH, cfg.HeadDim = D, cfg.Causal = true, cfg.KVHeadCount = KV;
    be().MultiHeadAttentionPacked(cfg, dq.data, dk.data, dv.data, o.data, doff.data, nullptr, B, rows, rows, DType::BFloat16);
    be().CheckStatus();
    std::vector<float> want;
    for (int64_t b = 0; b < B; ++b)
        for (int32_t t = 0; t < lens[b]; ++t) {
            auto row = attend(&q[(off[b] + t) * QH * D], &k[off[b] * KV * D], &v[off[b] * KV * D], t + 1);
            want.insert(want.end(), row.begin(), row.end());
        }
    double e = normwise(download_f32(o, DType::BFloat16), want);
    EXPECT(e <= 1e-2, "packed attention: normwise %.3g", e);

    // one token more each, attended over the 4-bit pages
    std::vector<int32_t> pos1, ids1, slots1, ctx;
    for (int64_t b = 0; b < B; ++b) {
        pos1.push_back(lens[b]);
        ids1.push_back(c.table[b * per + lens[b] / PS]);
        slots1.push_back(lens[b] % PS);
        ctx.push_back(lens[b] + 1);
    }
    auto bits1 = encode(normal(702, B * W), DType::BFloat16);
    std::vector<float> q1, k1, v1;
    split(decode(bits1, DType::BFloat16, B * W), B, q1, k1, v1);
    Tensor dq1 = append(c, upload(bits1, {B, W}, DType::BFloat16), B, pos1, ids1, slots1);
    k1 = rotated(k1, KV, pos1);
    const int64_t most = *std::max_element(ctx.begin(), ctx.end());
    const size_t ws = be().PagedInt4WorkspaceBytes(B, 1, QH, KV, D, most);
    Tensor dws = be().AllocateTensor({(int64_t)ws}, DType::Int8), o1 = be().AllocateTensor({B, QH * D}, DType::BFloat16);
    Tensor dt = upload(c.table, {B, per}, DType::Int32), dc = upload(ctx, {B}, DType::Int32);
    be().PagedInt4Attention(dq1.data, c.k.data, c.v.data, c.kp.data, c.vp.data, dt.data, dc.data, B, 1, per, PS, c.pages, QH, KV, D, G,
                            most, DType::BFloat16, o1.data, dws.data, ws);
    auto q1r = download_f32(dq1, DType::BFloat16);
    std::vector<float> want1;
    for (int64_t b = 0; b < B; ++b) {
        auto kg = gathered(c, c.k, c.kp, b, ctx[b]), vg = gathered(c, c.v, c.vp, b, ctx[b]);
        // what was stored: off by half a step of the group, by the roundings of its scale and offset
        // (2^-11 of 15 / 2 steps and of the largest value) and by f32's
        for (int which = 0; which < 2; ++which) {
            const std::vector<float> &got = which ? vg : kg, &prompt = which ? v : k, &last = which ? v1 : k1;
            for (int32_t t = 0; t < ctx[b]; ++t)
                for (int64_t g = 0; g < KV * D / G; ++g) {
                    const float *src = t < lens[b] ? &prompt[(off[b] + t) * KV * D + g * G] : &last[b * KV * D + g * G];
                    const float lo = *std::min_element(src, src + G), hi = *std::max_element(src, src + G);
                    const double step = (hi - lo) / 15.0, big = std::max(std::fabs(lo), std::fabs(hi));
                    const double bound = step * (0.5 + 16 * 0x1p-11) + big * 0x1p-10 + 1e-5;
                    for (int64_t i = 0; i < G; ++i) {
                        const double off_by = std::fabs((double)got[t * KV * D + g * G + i] - src[i]);
                        EXPECT(off_by <= bound, "%s of token %d, group %d: off by %.4g, bound %.4g", which ? "value" : "key", t, (int)g,
                               off_by, bound);
                    }
                }
        }
        auto row = attend(&q1r[b * QH * D], kg.data(), vg.data(), ctx[b]);
        want1.insert(want1.end(), row.begin(), row.end());
    }
    e = normwise(download_f32(o1, DType::BFloat16), want1);
    EXPECT(e <= 1e-2, "4-bit attention: normwise %.3g", e);
}

CASE(errors_reach_the_caller) {
    Cache c(1, 2);
    Tensor x = upload(encode(normal(703, (QH + 2 * KV) * D), DType::BFloat16), {1, (QH + 2 * KV) * D}, DType::BFloat16);
    bool thrown = false;
    try {
        append(c, x, 1, {0}, {(int32_t)c.pages}, {0});   // a page that is not there
    } catch (const Error &) {
        thrown = true;
    }
    EXPECT(thrown, "a page id past the pool");
    be().CheckStatus();   // reported once
    MultiHeadAttentionConfig cfg;
    cfg.NumHeads = 8, cfg.HeadDim = D, cfg.KVHeadCount = 3;
    thrown = false;
    try {
        be().MultiHeadAttentionPacked(cfg, x.data, x.data, x.data, x.data, x.data, nullptr, 1, 1, 1, DType::BFloat16);
    } catch (const Error &) {
        thrown = true;
    }
    EXPECT(thrown, "heads that the kv heads do not divide");
    thrown = false;
    try {
        be().PagedInt4Attention(x.data, c.k.data, c.v.data, c.kp.data, c.vp.data, x.data, x.data, 1, 1, 2, PS, c.pages, QH, KV, D, G, 20,
                                DType::BFloat16, x.data, x.data, 16);
    } catch (const Error &) {
        thrown = true;
    }
    EXPECT(thrown, "a workspace of 16 bytes");
}

int main(int argc, char **argv) {
    int count = 0;
    if (puter_hip_device_count(&count) != 0 || count < 1) {
        std::printf("no GPU\n");
        return 2;
    }
    return check::run_all(argc, argv);
}
