// Host-side check, on the library's own source (no device), of what a prompt,
// a tree or an 8-bit step is cut into.  Without arguments: over many shapes
// and calls, the kernels exist, the records and counters fit the workspace and
// the tiles cover the tokens.  With "plan": answers calls read from its input,
// one a line: q heads, KV heads, head_dim, 8-bit cache (0 or 1), step (0 or
// 1), sequences, rows of the packed arrays, a sequence's most tokens, the last
// position -> rows of a tile, one launch (1) or two (0), chunks, spread over
// the XCDs.  With "refuse": host-pointer calls whose begins go backwards.
// Built and run by tests/test_many_rules.py.
#include "checkpoint.cpp"
#include "leap_hip_attention.hip"

#include <cstdlib>

#define REQUIRE(c, ...)                                      \
    do {                                                     \
        if (!(c)) {                                          \
            std::printf("line %d: %s: ", __LINE__, #c);      \
            std::printf(__VA_ARGS__);                        \
            std::printf("\n");                               \
            std::exit(1);                                    \
        }                                                    \
    } while (0)

namespace {

leap_hip_attention handle(int n_heads, int n_kv_heads, int head_dim, int seq_len, int max_batch, bool q8)
{
    leap_hip_attention h;
    h.cfg = leap_hip_attention_config{};
    h.cfg.n_layers = h.cfg.layer_end = 1;
    h.cfg.n_heads = n_heads;
    h.cfg.n_kv_heads = n_kv_heads;
    h.cfg.head_dim = head_dim;
    h.cfg.seq_len = seq_len;
    h.cfg.max_batch = max_batch;
    h.group = n_heads / n_kv_heads;
    h.q_dim = n_heads * head_dim;
    h.kv_dim = n_kv_heads * head_dim;
    h.n_cu = 256;
    h.q8kv = q8;
    return h;
}

void check_plan(const leap_hip_attention &h, bool step, int n_seq, int n_tokens, int max_tokens, int max_pos)
{
    const ManyPlan p = many_plan(&h, step, n_seq, n_tokens, max_tokens, max_pos);
#define CALL "%d/%d/%d q8 %d step %d: %d sequences, %d rows, %d a sequence, to %d", h.cfg.n_heads, h.cfg.n_kv_heads, \
             h.cfg.head_dim, h.q8kv, step, n_seq, n_tokens, max_tokens, max_pos
    REQUIRE(p.fn.attention && p.fn.append, CALL);
    REQUIRE(!p.spread || p.fn.merge[0], CALL);
    REQUIRE(p.splits >= 1 && p.splits <= leap::kManySplits, CALL);
    REQUIRE((long long)p.chunk * p.splits > max_pos, CALL);
    REQUIRE(p.splits == 1 || (size_t)p.groups * p.splits * p.fn.rows <= kManyRecords, CALL);
    REQUIRE(p.splits == 1 || (size_t)p.groups <= kManyCounters, CALL);
    REQUIRE(p.wgs >= p.groups * p.splits && p.wgs > 0, CALL);
    // (as many tiles as a batch of full sequences and a rest has)
    const long long full = max_tokens ? n_tokens / max_tokens : 0, rest = max_tokens ? n_tokens % max_tokens : 0;
    const auto tiles = [&](long long n) { return (n * h.group + p.fn.rows - 1) / p.fn.rows; };
    const long long seqs = std::min<long long>(full, n_seq);
    REQUIRE(p.slots >= seqs * tiles(max_tokens) + (seqs < n_seq ? tiles(rest) : 0), CALL);
    REQUIRE(!p.fused || max_tokens <= (p.fn.rows == leap::kWideRows ? leap::kTreeMax : leap::kSmallNew), CALL);
#undef CALL
}

int sweep()
{
    const int shapes[][3] = {{32, 8, 128}, {32, 4, 64}, {32, 32, 128}, {64, 8, 128}, {4, 4, 64}, {6, 3, 128}, {32, 2, 128}, {3, 1, 64}};
    for (const auto &s : shapes)
        for (int q8 = 0; q8 < 2; q8++) {
            const leap_hip_attention h = handle(s[0], s[1], s[2], 131072, 256, q8);
            for (int n_seq : {1, 2, 7, 32, 65, 256})
                for (int last : {0, 1, 63, 255, 256, 1000, 4095, 8192, 65535, 131071}) {
                    if (q8) check_plan(h, true, n_seq, n_seq, 1, last);
                    for (int most : {1, 2, 8, 31, 32, 33, 64, 65, 500, 2048, 8192}) {
                        if (most > last + 1) break;
                        for (int all : {most, std::min(n_seq * most, most + n_seq), n_seq * most}) check_plan(h, false, n_seq, all, most, last);
                    }
                }
        }
    return 0;
}

int plans()
{
    int nh, nkv, hd, q8, step, n_seq, n_tokens, max_tokens, max_pos;
    while (std::scanf("%d %d %d %d %d %d %d %d %d", &nh, &nkv, &hd, &q8, &step, &n_seq, &n_tokens, &max_tokens, &max_pos) == 9) {
        const leap_hip_attention h = handle(nh, nkv, hd, max_pos + 1, n_seq, q8);
        const ManyPlan p = many_plan(&h, step, n_seq, n_tokens, max_tokens, max_pos);
        std::printf("%d %d %d %d\n", p.fn.rows, p.fused, p.splits, p.spread);
    }
    return 0;
}

// begins that go backwards: the rows of the arrays are begin's last, and a
// tree's parents behind them are none of its.
int refusals()
{
    leap_hip_attention h = handle(8, 2, 128, 64, 2, false);
    const int begin[] = {0, 5, 4}, pos[] = {0, 0};
    const int parent[] = {-1, 0, 1, 2, /* not the caller's: */ 77};
    float x[4];
    REQUIRE(leap_hip_attention_tree(&h, 0, 2, begin, pos, parent, x, x, x, x) == -EINVAL, "tree");
    REQUIRE(h.err.find("below") != std::string::npos, "%s", h.err.c_str());
    REQUIRE(leap_hip_attention_prompt(&h, 0, 2, begin, pos, x, x, x, x) == -EINVAL, "prompt");
    REQUIRE(h.err.find("below") != std::string::npos, "%s", h.err.c_str());
    return 0;
}

}  // namespace

int main(int argc, char **argv)
{
    const std::string what = argc > 1 ? argv[1] : "";
    return what == "plan" ? plans() : what == "refuse" ? refusals() : sweep();
}
