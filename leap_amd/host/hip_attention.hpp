// C++20 engine-side wrapper of the leap_hip_attention C ABI.
//
// This is the thin layer a LEAP engine (src/inference/FloatTransformer.cpp or
// QuantizedTransformer.cpp) keeps around the shim: it owns one handle, turns
// negative status codes into std::runtime_error the way the engine reports
// its own failures (TransformerFactory.cpp:59-135 throws runtime_error), and
// exposes the attention block of run_layer (FloatTransformer.cpp:396-662) as
// one call.
#pragma once

#include <cerrno>
#include <cstddef>
#include <cstdint>
#include <optional>
#include <span>
#include <stdexcept>
#include <string>
#include <utility>

#include "leap_hip_attention.h"

namespace leap {

class HipAttention {
public:
    struct Dims {
        int n_layers, layer_begin, layer_end, n_heads, n_kv_heads, head_dim, seq_len;
        float rope_theta = 500000.0f;  // FloatTransformer.cpp:65
        int max_batch = 1;
        int device = 0;
        bool cache_q8 = false;  // an 8-bit cache (leap_hip_attention_create_q8kv)
    };

    explicit HipAttention(const Dims &d)
    {
        const leap_hip_attention_config c{d.n_layers, d.layer_begin, d.layer_end, d.n_heads,
                                          d.n_kv_heads, d.head_dim,    d.seq_len,   d.rope_theta,
                                          d.max_batch,  d.device};
        check(d.cache_q8 ? leap_hip_attention_create_q8kv(&c, &h_) : leap_hip_attention_create(&c, &h_), nullptr);
        q_dim_ = d.n_heads * d.head_dim;
        kv_dim_ = d.n_kv_heads * d.head_dim;
    }
    HipAttention(const HipAttention &) = delete;
    HipAttention &operator=(const HipAttention &) = delete;
    HipAttention(HipAttention &&o) noexcept : h_(std::exchange(o.h_, nullptr)), q_dim_(o.q_dim_), kv_dim_(o.kv_dim_) {}
    ~HipAttention() { leap_hip_attention_destroy(h_); }

    // The attention block of run_layer(l, pos, x): q is s->q (pre-RoPE),
    // k_new / v_new the k and v GEMV outputs, out receives s->xb.
    void step(int layer, int pos, std::span<const float> q, std::span<const float> k_new,
              std::span<const float> v_new, std::span<float> out)
    {
        if ((int)q.size() != q_dim_ || (int)out.size() != q_dim_ || (int)k_new.size() != kv_dim_ ||
            (int)v_new.size() != kv_dim_)
            throw std::invalid_argument("HipAttention::step: buffer sizes do not match the model");
        check(leap_hip_attention_step(h_, layer, pos, q.data(), k_new.data(), v_new.data(), out.data()), h_);
    }

    // step() over whole prompts: tokens begin[i] .. begin[i+1] - 1 of the packed
    // rows are sequence i's, from position pos[i] on.
    void prompt(int layer, std::span<const int> begin, std::span<const int> pos, std::span<const float> q,
                std::span<const float> k_new, std::span<const float> v_new, std::span<float> out)
    {
        check_rows("prompt", begin, pos, q, k_new, v_new, out);
        check(leap_hip_attention_prompt(h_, layer, (int)pos.size(), begin.data(), pos.data(), q.data(), k_new.data(),
                                        v_new.data(), out.data()),
              h_);
    }

    // The same of drafted trees: parent of each node within its tree, or -1.
    void tree(int layer, std::span<const int> begin, std::span<const int> pos, std::span<const int> parent,
              std::span<const float> q, std::span<const float> k_new, std::span<const float> v_new, std::span<float> out)
    {
        check_rows("tree", begin, pos, q, k_new, v_new, out);
        if (parent.size() * (size_t)q_dim_ != q.size())
            throw std::invalid_argument("HipAttention::tree: one parent a row");
        check(leap_hip_attention_tree(h_, layer, (int)pos.size(), begin.data(), pos.data(), parent.data(), q.data(),
                                      k_new.data(), v_new.data(), out.data()),
              h_);
    }

    // The accepted paths' rows ([pos.size()][max_path] nodes, ended by -1) to
    // pos[i], pos[i] + 1, ..., in every held layer.
    void tree_keep(std::span<const int> pos, std::span<const int> path, int max_path)
    {
        if (max_path < 0 || path.size() != pos.size() * (size_t)max_path)
            throw std::invalid_argument("HipAttention::tree_keep: path must hold max_path nodes a sequence");
        check(leap_hip_attention_tree_keep(h_, (int)pos.size(), pos.data(), path.data(), max_path), h_);
    }

    // Weights of one held layer for block(): the layer's slices of
    // FloatTransformerWeights (FloatTransformer.h:9-22), row-major.
    void set_layer_weights(int layer, std::span<const float> rms_att, std::span<const float> wq,
                           std::span<const float> wk, std::span<const float> wv, std::span<const float> wo)
    {
        const size_t dim = (size_t)q_dim_, kv = (size_t)kv_dim_;
        if (rms_att.size() != dim || wq.size() != dim * dim || wk.size() != kv * dim || wv.size() != kv * dim ||
            wo.size() != dim * dim)
            throw std::invalid_argument("HipAttention::set_layer_weights: weight sizes do not match the model");
        check(leap_hip_attention_set_layer_weights(h_, layer, rms_att.data(), wq.data(), wk.data(), wv.data(),
                                                   wo.data()),
              h_);
    }

    // The int8 engine's weights of one held layer: each projection as the
    // reference's QuantizedTensor (QuantizedTransformer.h:9-12), int8 values
    // [d][n] and one scale per group of group_size values.
    struct QTensor {
        std::span<const int8_t> q;
        std::span<const float> s;
    };
    void set_layer_weights_q8(int layer, int group_size, std::span<const float> rms_att, QTensor wq, QTensor wk,
                              QTensor wv, QTensor wo)
    {
        const size_t dim = (size_t)q_dim_, kv = (size_t)kv_dim_;
        const auto ok = [&](const QTensor &t, size_t rows) {
            return group_size > 0 && t.q.size() == rows * dim && t.s.size() == rows * dim / (size_t)group_size;
        };
        if (rms_att.size() != dim || !ok(wq, dim) || !ok(wk, kv) || !ok(wv, kv) || !ok(wo, dim))
            throw std::invalid_argument("HipAttention::set_layer_weights_q8: weight sizes do not match the model");
        check(leap_hip_attention_set_layer_weights_q8(h_, layer, group_size, rms_att.data(), wq.q.data(),
                                                      wq.s.data(), wk.q.data(), wk.s.data(), wv.q.data(),
                                                      wv.s.data(), wo.q.data(), wo.s.data()),
              h_);
    }

    // run_layer(l, pos, x) from its start to the attention residual
    // (FloatTransformer.cpp:394-683): x += Wo . attention(Wq/Wk/Wv . rmsnorm(x)).
    void block(int layer, int pos, std::span<float> x)
    {
        if ((int)x.size() != q_dim_)
            throw std::invalid_argument("HipAttention::block: x must hold dim floats");
        check(leap_hip_attention_block(h_, layer, pos, x.data()), h_);
    }

    // The same with x in device memory (16-byte aligned), enqueued on `stream`.
    void block_async(int layer, int pos, float *x_dev, void *stream)
    {
        check(leap_hip_attention_block_async(h_, layer, pos, x_dev, stream), h_);
    }

    // ---- the stage hand-off of a pipeline (FloatTransformer.cpp:775-788, 925-939)

    // PacketHeader (Transformer.h:25-28).
    struct PacketHeader {
        int pos, flags;
    };
    size_t packet_bytes() const { return LEAP_HIP_ATTENTION_PACKET_HEADER_BYTES + sizeof(float) * (size_t)q_dim_; }

    // A received packet's x into the device residual stream x_dev; its header,
    // or nothing for a control packet (the transport's business).  Enqueued on
    // `stream`; a null stream waits for the copy.
    std::optional<PacketHeader> upload_packet(std::span<const std::byte> packet, float *x_dev, void *stream = nullptr)
    {
        PacketHeader hd{};
        const int rc = leap_hip_attention_packet_upload(h_, packet.data(), packet.size(), x_dev, &hd.pos, &hd.flags,
                                                        stream);
        if (rc == 1) return std::nullopt;
        check(rc, h_);
        return hd;
    }

    // The packet {header, x_dev} for the next stage; its values are in place
    // once `stream` has passed the copy (at return for a null stream).
    void download_packet(const float *x_dev, PacketHeader hd, std::span<std::byte> packet, void *stream = nullptr)
    {
        check(leap_hip_attention_packet_download(h_, x_dev, hd.pos, hd.flags, packet.data(), packet.size(), stream),
              h_);
    }

    // worker_loop forwards after its layers unless it is the tail and no
    // reply is wanted (FloatTransformer.cpp:937).
    static bool forwards(bool is_tail, int flags) { return !is_tail || flags == LEAP_HIP_ATTENTION_FLAG_NEED_REPLY; }

    // Every held layer's attention weights from a checkpoint file
    // (Transformer::create's format, TransformerFactory.cpp:59-135).
    void load_checkpoint(const std::string &path) { check(leap_hip_attention_load_checkpoint(h_, path.c_str()), h_); }

    // The header of a checkpoint file.
    static leap_hip_attention_checkpoint checkpoint_read(const std::string &path)
    {
        leap_hip_attention_checkpoint c{};
        if (int rc = leap_hip_attention_checkpoint_read(path.c_str(), &c))
            throw std::runtime_error("leap_hip_attention: cannot read checkpoint " + path + " (status " +
                                     std::to_string(rc) + ")");
        return c;
    }

    // clear_kv_cache (FloatTransformer.cpp:74-77).
    void clear_kv_cache() { check(leap_hip_attention_clear(h_), h_); }

    void kv_download(int seq, int layer, int pos_begin, int pos_end, float *k, float *v)
    {
        check(leap_hip_attention_kv_download(h_, seq, layer, pos_begin, pos_end, k, v), h_);
    }

    leap_hip_attention *handle() const { return h_; }

private:
    static void check(int rc, const leap_hip_attention *h)
    {
        if (rc != 0)
            throw std::runtime_error(std::string("leap_hip_attention: ") + leap_hip_attention_last_error(h) +
                                     " (status " + std::to_string(rc) + ")");
    }

    void check_rows(const char *what, std::span<const int> begin, std::span<const int> pos, std::span<const float> q,
                    std::span<const float> k_new, std::span<const float> v_new, std::span<float> out) const
    {
        const size_t n = q.size() / (size_t)q_dim_;
        if (pos.empty() || begin.size() != pos.size() + 1 || begin.back() < 0 || (size_t)begin.back() > n ||
            q.size() != n * (size_t)q_dim_ || out.size() != q.size() || k_new.size() != n * (size_t)kv_dim_ ||
            v_new.size() != k_new.size())
            throw std::invalid_argument(std::string("HipAttention::") + what + ": buffer sizes do not match");
    }

    leap_hip_attention *h_ = nullptr;
    int q_dim_ = 0, kv_dim_ = 0;
};

// A cache of pages (leap_hip_attention_pages): sequences of a batch that share
// rows and hold no more memory than they use.
class HipPages {
public:
    struct Dims {
        HipAttention::Dims model;  // (cache_q8: pages of 8-bit rows)
        int n_pages;
        int page_rows = 16;   // 16, 32, 64 or 128
        bool bounds = false;  // step_sparse needs them
    };

    explicit HipPages(const Dims &d)
    {
        const HipAttention::Dims &m = d.model;
        const leap_hip_attention_pages_config c{{m.n_layers, m.layer_begin, m.layer_end, m.n_heads, m.n_kv_heads, m.head_dim,
                                                 m.seq_len, m.rope_theta, m.max_batch, m.device},
                                                d.page_rows, d.n_pages, m.cache_q8, d.bounds};
        check(leap_hip_attention_pages_create(&c, &p_), nullptr);
        q_dim_ = m.n_heads * m.head_dim;
        kv_dim_ = m.n_kv_heads * m.head_dim;
        n_kv_heads_ = m.n_kv_heads;
    }
    HipPages(const HipPages &) = delete;
    HipPages &operator=(const HipPages &) = delete;
    HipPages(HipPages &&o) noexcept
        : p_(std::exchange(o.p_, nullptr)), q_dim_(o.q_dim_), kv_dim_(o.kv_dim_), n_kv_heads_(o.n_kv_heads_)
    {
    }
    ~HipPages() { leap_hip_attention_pages_destroy(p_); }

    // Pages of its own for rows [begin[i], end[i]) of each sequence; false, with
    // nothing changed, where the pool has too few.
    bool reserve(std::span<const int> begin, std::span<const int> end)
    {
        same(begin.size(), end.size(), "reserve: begin and end");
        const int rc = leap_hip_attention_pages_reserve(p_, (int)begin.size(), begin.data(), end.data());
        if (rc == -ENOMEM) return false;
        check(rc, p_);
        return true;
    }
    // Sequence i takes the pages of the first rows[i] rows of parent[i] (empty: its own).
    void fork(std::span<const int> parent, std::span<const int> rows)
    {
        if (!parent.empty()) same(parent.size(), rows.size(), "fork: parent and rows");
        check(leap_hip_attention_pages_fork(p_, (int)rows.size(), parent.empty() ? nullptr : parent.data(), rows.data()), p_);
    }
    // The pages in use to the front of the pool; how many there are.
    int compact()
    {
        int used = 0;
        check(leap_hip_attention_pages_compact(p_, &used), p_);
        return used;
    }

    // One token of each sequence, at pos[i], whose row is reserved.
    void step(int layer, std::span<const int> pos, std::span<const float> q, std::span<const float> k_new,
              std::span<const float> v_new, std::span<float> out)
    {
        check_rows(pos, q, k_new, v_new, out);
        check(leap_hip_attention_pages_step(p_, layer, (int)pos.size(), pos.data(), q.data(), k_new.data(), v_new.data(), out.data()), p_);
    }
    // The same over at most `keep` pages for each KV head; picked: empty, or [pos.size()][n_kv_heads][keep].
    void step_sparse(int layer, std::span<const int> pos, int keep, std::span<const float> q, std::span<const float> k_new,
                     std::span<const float> v_new, std::span<float> out, std::span<int> picked = {})
    {
        check_rows(pos, q, k_new, v_new, out);
        if (!picked.empty()) same(picked.size(), pos.size() * (size_t)n_kv_heads_ * (size_t)(keep > 0 ? keep : 0), "step_sparse: picked");
        check(leap_hip_attention_pages_step_sparse(p_, layer, (int)pos.size(), pos.data(), keep, q.data(), k_new.data(), v_new.data(),
                                                   out.data(), picked.empty() ? nullptr : picked.data()),
              p_);
    }

    // Rows [begin, begin + k.size() / kv_dim) of a sequence, k as it is stored (after rotation).
    void write(int seq, int layer, int begin, std::span<const float> k, std::span<const float> v)
    {
        check_kv(k.size(), v.size(), "write");
        check(leap_hip_attention_pages_write(p_, seq, layer, begin, begin + (int)(k.size() / (size_t)kv_dim_), k.data(), v.data()), p_);
    }
    void read(int seq, int layer, int begin, std::span<float> k, std::span<float> v)
    {
        check_kv(k.size(), v.size(), "read");
        check(leap_hip_attention_pages_read(p_, seq, layer, begin, begin + (int)(k.size() / (size_t)kv_dim_), k.data(), v.data()), p_);
    }

    // The `beams` best continuations of each group of beams: logits [score.size()][vocab].
    void beam_select(int beams, std::span<const float> logits, std::span<const float> score, std::span<int> parent,
                     std::span<int> token, std::span<float> best)
    {
        const size_t n = score.size();
        same(parent.size(), n, "beam_select: parent");
        same(token.size(), n, "beam_select: token");
        same(best.size(), n, "beam_select: best");
        if (n == 0 || beams <= 0 || n % (size_t)beams || logits.size() % n)
            throw std::invalid_argument("HipPages::beam_select: sizes are no groups of beams");
        check(leap_hip_attention_pages_beam_select(p_, (int)(n / (size_t)beams), beams, (int)(logits.size() / n), logits.data(),
                                                   score.data(), parent.data(), token.data(), best.data()),
              p_);
    }

    void clear() { check(leap_hip_attention_pages_clear(p_), p_); }
    leap_hip_attention_pages *handle() { return p_; }

private:
    static void same(size_t a, size_t b, const char *what)
    {
        if (a != b) throw std::invalid_argument(std::string("HipPages::") + what + ": sizes differ");
    }
    void check_kv(size_t k, size_t v, const char *what) const
    {
        same(k, v, what);
        same(k % (size_t)kv_dim_, 0, what);
    }
    void check_rows(std::span<const int> pos, std::span<const float> q, std::span<const float> k, std::span<const float> v,
                    std::span<const float> out) const
    {
        same(q.size(), pos.size() * (size_t)q_dim_, "step: q");
        same(out.size(), q.size(), "step: out");
        same(k.size(), pos.size() * (size_t)kv_dim_, "step: k_new");
        same(v.size(), k.size(), "step: v_new");
    }
    static void check(int rc, leap_hip_attention_pages *p)
    {
        if (rc != 0) throw std::runtime_error(std::string("leap_hip_attention_pages: ") + leap_hip_attention_pages_last_error(p));
    }

    leap_hip_attention_pages *p_ = nullptr;
    int q_dim_ = 0, kv_dim_ = 0, n_kv_heads_ = 0;
};

}  // namespace leap
