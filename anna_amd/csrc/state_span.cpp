// Layout of the packed tokens of sequences that continue states (anna_mi_state_span).
#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

#include "delta.hpp"

namespace anna {

// Sizes of a span, and with `words` its content.  Sequences of at most STEP_TOKENS tokens are taken token by
// token, longer ones ("chains") in chunks.
static int lay_out(int64_t n, const int32_t* slots, const int64_t* counts, const int32_t* fresh, anna_mi_state_span* s,
                   int32_t* words) {
  ANNA_CHECK(s != nullptr, "state span: null span");
  ANNA_CHECK(n >= 0 && n <= INT32_MAX / 4, "state span: %lld sequences", (long long)n);
  ANNA_CHECK(n == 0 || (slots && counts), "state span: null slots or counts");
  int64_t tokens = 0, steps = 0, chains = 0, chunks = 0, longest = 0, max_slot = -1;
  for (int64_t i = 0; i < n; i++) {
    ANNA_CHECK(slots[i] >= -1, "state span: slot %d of sequence %lld", (int)slots[i], (long long)i);
    ANNA_CHECK(counts[i] >= 0 && counts[i] <= INT32_MAX, "state span: sequence %lld of %lld tokens", (long long)i, (long long)counts[i]);
    tokens += counts[i];
    ANNA_CHECK(tokens <= INT32_MAX - 4095, "state span: more than 2^31 - 4096 tokens");  // kernels count a little further
    max_slot = std::max<int64_t>(max_slot, slots[i]);
    if (counts[i] > STEP_TOKENS) {
      chains++;
      const int64_t own = (counts[i] + CHUNK - 1) / CHUNK;
      chunks += own;
      longest = std::max(longest, own);
    } else if (counts[i] > 0) {
      steps++;
    }
  }
  try {
    std::vector<int32_t> used(slots, slots + n);
    std::sort(used.begin(), used.end());
    for (int64_t i = 1; i < n; i++)
      ANNA_CHECK(used[i] != used[i - 1] || used[i] < 0, "state span: slot %d is named twice", (int)used[i]);
  } catch (const std::bad_alloc&) {
    set_error("state span: out of host memory");
    return ANNA_MI_EINVAL;
  }
  const int64_t total = 4 * n + 4 * steps + 8 * chains + 4 * chunks + tokens;
  if (words) {
    ANNA_CHECK(s->sequences == n && s->tokens == tokens && s->steps == steps && s->chains == chains && s->chunks == chunks && s->longest == longest &&
                   s->words == std::max<int64_t>(1, total),
               "state span: filled with other counts than it was planned for");
    s->max_slot = max_slot;
    int32_t* step = words + 4 * n;
    int32_t* const chain = step + 4 * steps;
    int32_t* chunk = chain + 8 * chains;
    int32_t* owner = chunk + 4 * chunks;
    int32_t first = 0, first_chunk = 0;
    for (int64_t i = 0, c = 0; i < n; i++) {
      const int32_t count = (int32_t)counts[i];
      const int32_t record[8] = {slots[i], first, count, fresh && fresh[i] ? 1 : 0, first_chunk, 0, 0, 0};
      std::copy(record, record + 4, words + 4 * i);
      if (count > STEP_TOKENS) {
        std::copy(record, record + 8, chain + 8 * c++);
        for (int32_t at = 0; at < count; at += CHUNK, first_chunk++) {
          const int32_t part[4] = {slots[i], first + at, std::min(CHUNK, count - at), 0};
          chunk = std::copy(part, part + 4, chunk);
        }
      } else if (count > 0) {
        step = std::copy(record, record + 4, step);
      }
      owner = std::fill_n(owner, count, (int32_t)i);
      first += count;
    }
    // the longest chains first: their workgroups start first, and the short ones fill what is left
    struct Record {
      int32_t v[8];
    };
    Record* const sorted = (Record*)chain;
    std::stable_sort(sorted, sorted + chains, [](const Record& a, const Record& b) { return a.v[2] > b.v[2]; });
    if (total == 0) words[0] = 0;
    return ANNA_MI_OK;
  }
  s->sequences = n;
  s->tokens = tokens;
  s->words = std::max<int64_t>(1, total);
  s->steps = steps;
  s->chains = chains;
  s->chunks = chunks;
  s->longest = longest;
  s->max_slot = max_slot;
  s->least_slots = INT64_MAX;
  return ANNA_MI_OK;
}

// Calls of several threads may take one span, without a lock of theirs, while another names its next slots: what a span
// promises a pool (slots below max_slot) and what pools it was taken with change together.
static std::mutex span_lock;

int span_take(anna_mi_state_span* s, int64_t slots, const char* what) {
  const std::lock_guard<std::mutex> held(span_lock);
  ANNA_CHECK(s->max_slot < slots, "%s: slot %lld of a state of %lld", what, (long long)s->max_slot, (long long)slots);
  s->least_slots = std::min(s->least_slots, slots);
  return ANNA_MI_OK;
}

}  // namespace anna

extern "C" {

int anna_mi_state_span_plan(int64_t n, const int32_t* slots, const int64_t* counts, const int32_t* fresh,
                            anna_mi_state_span* span) {
  return anna::lay_out(n, slots, counts, fresh, span, nullptr);
}

int anna_mi_state_span_fill(int64_t n, const int32_t* slots, const int64_t* counts, const int32_t* fresh,
                            anna_mi_state_span* span, int32_t* words) {
  ANNA_CHECK(words != nullptr, "state span: null words");
  return anna::lay_out(n, slots, counts, fresh, span, words);
}

int anna_mi_state_span_refill(anna_mi_state_span* span, const anna_mi_state_span* plan) {
  ANNA_CHECK(span != nullptr && plan != nullptr, "state span: null span or plan");
  ANNA_CHECK(span->sequences == plan->sequences && span->words == plan->words && span->tokens == plan->tokens && span->steps == plan->steps &&
                 span->chains == plan->chains && span->chunks == plan->chunks && span->longest == plan->longest,
             "state span: filled with other counts than it was planned for");
  const std::lock_guard<std::mutex> held(anna::span_lock);
  ANNA_CHECK(plan->max_slot < span->least_slots, "slot %lld: the span was used with states of %lld slots", (long long)plan->max_slot,
             (long long)span->least_slots);
  span->max_slot = plan->max_slot;
  return ANNA_MI_OK;
}

int64_t anna_mi_sizeof_state_span(void) { return (int64_t)sizeof(anna_mi_state_span); }
int64_t anna_mi_sizeof_gated_delta_args(void) { return (int64_t)sizeof(anna_mi_gated_delta_args); }
int64_t anna_mi_sizeof_rms_norm_args(void) { return (int64_t)sizeof(anna_mi_rms_norm_args); }

}  // extern "C"
