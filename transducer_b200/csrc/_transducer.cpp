// pybind11 module `_transducer`: the Python <-> C++ boundary.
//
// Exposes the three functions of the reference's shim under the same names and
// keyword arguments (transducer/_transducer.cpp:9-148 -- pointers travel as integers
// obtained from tensor.data_ptr()), plus the entry points of transducer_b200.h that
// replace the torch-op arithmetic of transducer/torch_binding.py.  Failures surface as
// ValueError (invalid argument) or RuntimeError (CUDA), as pybind11 maps the
// reference's std::invalid_argument / std::runtime_error.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/transducer.h"
#include "../../include/transducer_b200.h"

namespace py = pybind11;
using namespace py::literals;
using addr = std::uintptr_t;

namespace {

template <typename T>
T* at(addr a) { return reinterpret_cast<T*>(a); }

void check(int rc) {
  if (rc == TB200_OK) return;
  if (rc == TB200_ERR_INVALID_ARGUMENT || rc == TB200_ERR_WORKSPACE)
    throw std::invalid_argument(tb200_last_error());
  throw std::runtime_error(tb200_last_error());
}

// A call that waits for the stream: other threads of the interpreter go on meanwhile (what is waited for may need them).
template <typename F>
int waiting(F&& call) {
  py::gil_scoped_release released;
  return call();
}

// Which indices of a checked call are beyond their tensors: bit 0 frames, parents or words, bit 1 positions.
class Beyond {
 public:
  explicit Beyond(bool wanted) {
    if (wanted) check(tb200_flags_take(&flags_));
  }
  Beyond(const Beyond&) = delete;
  Beyond& operator=(const Beyond&) = delete;
  ~Beyond() {   // (the call has failed; kernels of it may still run)
    int values[2];
    if (flags_) waiting([&] { return tb200_flags_wait(flags_, values); });
  }
  int* flags() const { return flags_; }
  int wait() {
    if (!flags_) return 0;
    int values[2], *flags = flags_;
    flags_ = nullptr;
    check(waiting([&] { return tb200_flags_wait(flags, values); }));
    return (values[0] ? 1 : 0) | (values[1] ? 2 : 0);
  }

 private:
  int* flags_ = nullptr;
};

}  // namespace

PYBIND11_MODULE(_transducer, m) {
  m.doc() = "sm_100a RNN-T loss / Viterbi kernels (drop-in for awni/transducer's _transducer)";

  // ---- reference-compatible trio -------------------------------------------------
  m.def("forward",
        [](addr e, addr p, addr costs, addr alphas, addr ln, addr labels, addr ilen, addr llen,
           int B, int T, int U, int V, int blank, bool use_cuda) {
          forward(at<const float>(e), at<const float>(p), at<float>(costs), at<float>(alphas),
                  at<const float>(ln), at<const int>(labels), at<const int>(ilen),
                  at<const int>(llen), B, T, U, V, blank, use_cuda);
        },
        "emissions"_a, "predictions"_a, "costs"_a, "alphas"_a, "logNorms"_a, "labels"_a,
        "input_lengths"_a, "label_lengths"_a, "batch_size"_a, "max_input_length"_a,
        "max_label_length"_a, "alphabet_size"_a, "blank"_a, "use_cuda"_a);

  m.def("backward",
        [](addr e, addr p, addr eg, addr pg, addr lg, addr alphas, addr ln, addr labels,
           addr ilen, addr llen, int B, int T, int U, int V, int blank, bool use_cuda) {
          backward(at<const float>(e), at<const float>(p), at<float>(eg), at<float>(pg),
                   at<float>(lg), at<const float>(alphas), at<const float>(ln),
                   at<const int>(labels), at<const int>(ilen), at<const int>(llen), B, T, U, V,
                   blank, use_cuda);
        },
        "emissions"_a, "predictions"_a, "egrads"_a, "pgrads"_a, "lngrads"_a, "alphas"_a,
        "logNorms"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a, "batch_size"_a,
        "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a, "blank"_a,
        "use_cuda"_a);

  m.def("viterbi",
        [](addr e, addr p, addr ln, addr labels, addr ilen, addr llen, int B, int T, int U,
           int V, int blank, bool use_cuda) {
          viterbi(at<const float>(e), at<const float>(p), at<const float>(ln), at<int>(labels),
                  at<const int>(ilen), at<const int>(llen), B, T, U, V, blank, use_cuda);
        },
        "emissions"_a, "predictions"_a, "log_norms"_a, "labels"_a, "input_lengths"_a,
        "label_lengths"_a, "batch_size"_a, "max_input_length"_a, "max_label_length"_a,
        "alphabet_size"_a, "blank"_a, "use_cuda"_a);

  // ---- fused path ------------------------------------------------------------------
  m.def("set_stream", [](addr s) { check(tb200_set_stream(at<void>(s))); }, "stream"_a);
  m.def("set_option", [](const char* k, int v) { check(tb200_set_option(k, v)); }, "key"_a,
        "value"_a);
  m.def("get_option", [](const char* k) { int v = 0; check(tb200_get_option(k, &v)); return v; },
        "key"_a);

  m.def("log_norms_workspace_bytes", &tb200_log_norms_workspace_bytes);
  m.def("loss_forward_workspace_bytes", &tb200_loss_forward_workspace_bytes);
  m.def("loss_backward_workspace_bytes", &tb200_loss_backward_workspace_bytes);
  m.def("viterbi_decode_workspace_bytes", &tb200_viterbi_decode_workspace_bytes);

  m.def("log_norms",
        [](addr e, addr p, addr ln, addr rowref, addr maxp, addr ilen, addr llen, int B, int T,
           int U, int V, addr ws, size_t wsBytes) {
          check(tb200_log_norms(at<const float>(e), at<const float>(p), at<float>(ln),
                                at<float>(rowref), at<float>(maxp), at<const int>(ilen),
                                at<const int>(llen), B, T, U, V, at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "log_norms"_a, "row_ref"_a, "max_p"_a,
        "input_lengths"_a, "label_lengths"_a, "batch_size"_a, "max_input_length"_a,
        "max_label_length"_a, "alphabet_size"_a, "workspace"_a, "workspace_bytes"_a);

  m.def("loss_saved_bytes", &tb200_loss_saved_bytes);

  m.def("loss_forward",
        [](addr e, addr p, addr labels, addr ilen, addr llen, addr costs, addr loss_sum,
           addr saved, size_t savedBytes, int B, int T, int U, int V, int blank, addr ws,
           size_t wsBytes) {
          check(tb200_loss_forward(at<const float>(e), at<const float>(p), at<const int>(labels),
                                   at<const int>(ilen), at<const int>(llen), at<float>(costs),
                                   at<float>(loss_sum), at<void>(saved), savedBytes, B, T, U, V,
                                   blank, at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a,
        "costs"_a, "loss_sum"_a, "saved"_a, "saved_bytes"_a, "batch_size"_a,
        "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a, "blank"_a, "workspace"_a,
        "workspace_bytes"_a);

  m.def("loss_score_workspace_bytes", &tb200_loss_score_workspace_bytes);

  m.def("loss_score",
        [](addr e, addr p, addr labels, addr ilen, addr llen, addr costs, addr loss_sum, int B, int T,
           int U, int V, int blank, addr ws, size_t wsBytes, bool bf16) {
          check(bf16 ? tb200_loss_score_bf16(at<const void>(e), at<const void>(p), at<const int>(labels),
                                             at<const int>(ilen), at<const int>(llen), at<float>(costs),
                                             at<float>(loss_sum), B, T, U, V, blank, at<void>(ws), wsBytes)
                     : tb200_loss_score(at<const float>(e), at<const float>(p), at<const int>(labels),
                                        at<const int>(ilen), at<const int>(llen), at<float>(costs),
                                        at<float>(loss_sum), B, T, U, V, blank, at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a,
        "costs"_a, "loss_sum"_a, "batch_size"_a, "max_input_length"_a, "max_label_length"_a,
        "alphabet_size"_a, "blank"_a, "workspace"_a, "workspace_bytes"_a, "bf16"_a);

  m.def("loss_forward_bf16",
        [](addr e, addr p, addr labels, addr ilen, addr llen, addr costs, addr loss_sum,
           addr saved, size_t savedBytes, int B, int T, int U, int V, int blank, addr ws,
           size_t wsBytes) {
          check(tb200_loss_forward_bf16(at<const void>(e), at<const void>(p),
                                        at<const int>(labels), at<const int>(ilen),
                                        at<const int>(llen), at<float>(costs), at<float>(loss_sum),
                                        at<void>(saved), savedBytes, B, T, U, V, blank,
                                        at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a,
        "costs"_a, "loss_sum"_a, "saved"_a, "saved_bytes"_a, "batch_size"_a,
        "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a, "blank"_a, "workspace"_a,
        "workspace_bytes"_a);

  m.def("loss_backward_bf16",
        [](addr e, addr p, addr labels, addr ilen, addr llen, addr saved, size_t savedBytes,
           addr deltas, addr eg, addr pg, int B, int T, int U, int V, int blank, addr ws,
           size_t wsBytes) {
          check(tb200_loss_backward_bf16(at<const void>(e), at<const void>(p),
                                         at<const int>(labels), at<const int>(ilen),
                                         at<const int>(llen), at<const void>(saved), savedBytes,
                                         at<const float>(deltas), at<void>(eg), at<void>(pg), B,
                                         T, U, V, blank, at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a,
        "saved"_a, "saved_bytes"_a, "deltas"_a, "egrads"_a, "pgrads"_a, "batch_size"_a,
        "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a, "blank"_a, "workspace"_a,
        "workspace_bytes"_a);

  m.def("loss_backward",
        [](addr e, addr p, addr labels, addr ilen, addr llen, addr saved, size_t savedBytes,
           addr deltas, addr eg, addr pg, int B, int T, int U, int V, int blank, addr ws,
           size_t wsBytes) {
          check(tb200_loss_backward(at<const float>(e), at<const float>(p),
                                    at<const int>(labels), at<const int>(ilen),
                                    at<const int>(llen), at<const void>(saved), savedBytes,
                                    at<const float>(deltas), at<float>(eg), at<float>(pg), B, T,
                                    U, V, blank, at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "labels"_a, "input_lengths"_a, "label_lengths"_a,
        "saved"_a, "saved_bytes"_a, "deltas"_a, "egrads"_a, "pgrads"_a, "batch_size"_a,
        "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a, "blank"_a, "workspace"_a,
        "workspace_bytes"_a);

  m.def("viterbi_decode",
        [](addr e, addr p, addr ilen, addr llen, addr labels, int B, int T, int U, int V,
           int blank, addr ws, size_t wsBytes) {
          check(tb200_viterbi_decode(at<const float>(e), at<const float>(p), at<const int>(ilen),
                                     at<const int>(llen), at<int>(labels), B, T, U, V, blank,
                                     at<void>(ws), wsBytes));
        },
        "emissions"_a, "predictions"_a, "input_lengths"_a, "label_lengths"_a, "labels"_a,
        "batch_size"_a, "max_input_length"_a, "max_label_length"_a, "alphabet_size"_a,
        "blank"_a, "workspace"_a, "workspace_bytes"_a);

  // ---- operators on single lattice nodes ---------------------------------------------
  // `scores`: (emissions, predictions, bf16, their strides by utterance and by frame resp. position)
  using Scores = std::tuple<addr, addr, bool, long long, long long, long long, long long>;
  using Sizes = std::tuple<int, int, int, int, int>;   // B, T, U, V, N
  m.attr("node_summary_scratch_bytes") = tb200_node_summary_scratch_bytes();
  // (greatest frame, position, listed word), after one synchronisation
  m.def("node_summary",
        [](addr frames, addr positions, long long nodes, addr words, long long word_count, addr scratch) {
          int most[3];
          check(waiting([&] {
            return tb200_node_summary(at<const int>(frames), at<const int>(positions), nodes, at<const int>(words),
                                      word_count, at<void>(scratch), most);
          }));
          return py::make_tuple(most[0], most[1], most[2]);
        },
        "frames"_a, "positions"_a, "nodes"_a, "words"_a, "word_count"_a, "scratch"_a);
  m.def("top_words",
        [](const Scores& s, addr frames, addr positions, addr words, addr logits, addr rest, const Sizes& n, int k,
           double temperature) {
          check(tb200_top_words(at<const void>(std::get<0>(s)), at<const void>(std::get<1>(s)), std::get<2>(s),
                                std::get<3>(s), std::get<4>(s), std::get<5>(s), std::get<6>(s),
                                at<const int>(frames), at<const int>(positions), at<int>(words), at<float>(logits),
                                at<float>(rest), std::get<0>(n), std::get<1>(n), std::get<2>(n), std::get<3>(n),
                                std::get<4>(n), k, temperature));
        },
        "scores"_a, "frames"_a, "positions"_a, "words"_a, "logits"_a, "rest"_a, "sizes"_a, "k"_a, "temperature"_a);
  m.def("sample_words",
        [](const Scores& s, addr frames, addr positions, addr uniforms, addr words, addr log_probs, const Sizes& n,
           double temperature, int top_k, double top_p, double min_p) {
          check(tb200_sample_words(at<const void>(std::get<0>(s)), at<const void>(std::get<1>(s)), std::get<2>(s),
                                   std::get<3>(s), std::get<4>(s), std::get<5>(s), std::get<6>(s),
                                   at<const int>(frames), at<const int>(positions), at<const float>(uniforms),
                                   at<int>(words), at<float>(log_probs), std::get<0>(n), std::get<1>(n),
                                   std::get<2>(n), std::get<3>(n), std::get<4>(n), temperature, top_k, top_p, min_p));
        },
        "scores"_a, "frames"_a, "positions"_a, "uniforms"_a, "words"_a, "log_probs"_a, "sizes"_a, "temperature"_a,
        "top_k"_a, "top_p"_a, "min_p"_a);
  m.def("distill_saved_bytes", &tb200_distill_saved_bytes);
  m.def("distill_backward_workspace_bytes", &tb200_distill_backward_workspace_bytes);
  m.def("distill_forward",
        [](const Scores& s, addr frames, addr positions, addr words, addr logits, addr rest, addr costs, addr saved,
           size_t saved_bytes, const Sizes& n, int k, double temperature) {
          check(tb200_distill_forward(at<const void>(std::get<0>(s)), at<const void>(std::get<1>(s)), std::get<2>(s),
                                      std::get<3>(s), std::get<4>(s), std::get<5>(s), std::get<6>(s),
                                      at<const int>(frames), at<const int>(positions), at<const int>(words),
                                      at<const float>(logits), at<const float>(rest), at<float>(costs),
                                      at<void>(saved), saved_bytes, std::get<0>(n), std::get<1>(n), std::get<2>(n),
                                      std::get<3>(n), std::get<4>(n), k, temperature));
        },
        "scores"_a, "frames"_a, "positions"_a, "words"_a, "logits"_a, "rest"_a, "costs"_a, "saved"_a,
        "saved_bytes"_a, "sizes"_a, "k"_a, "temperature"_a);
  m.def("distill_backward",
        [](const Scores& s, addr frames, addr positions, addr words, addr saved, size_t saved_bytes, addr weights,
           addr egrads, addr pgrads, const Sizes& n, int k, double temperature, addr ws,
           size_t ws_bytes) {
          check(tb200_distill_backward(at<const void>(std::get<0>(s)), at<const void>(std::get<1>(s)),
                                       std::get<2>(s), std::get<3>(s), std::get<4>(s), std::get<5>(s),
                                       std::get<6>(s), at<const int>(frames), at<const int>(positions),
                                       at<const int>(words), at<const void>(saved), saved_bytes,
                                       at<const float>(weights), at<void>(egrads), at<void>(pgrads),
                                       std::get<0>(n), std::get<1>(n), std::get<2>(n), std::get<3>(n),
                                       std::get<4>(n), k, temperature, at<void>(ws), ws_bytes));
        },
        "scores"_a, "frames"_a, "positions"_a, "words"_a, "saved"_a, "saved_bytes"_a, "weights"_a, "egrads"_a,
        "pgrads"_a, "sizes"_a, "k"_a, "temperature"_a, "workspace"_a, "workspace_bytes"_a);

  // ---- a beam search's step, words' embeddings -----------------------------------------
  m.def("extend_beams_workspace_bytes", &tb200_extend_beams_workspace_bytes);
  m.def("extend_beams",
        [](const Scores& s, addr frames, addr positions, addr scores, addr out_scores, addr parents, addr words,
           const Sizes& n, int width, bool validate, addr ws, size_t ws_bytes) {
          Beyond beyond(validate);
          check(tb200_extend_beams(at<const void>(std::get<0>(s)), at<const void>(std::get<1>(s)), std::get<2>(s),
                                   std::get<3>(s), std::get<4>(s), std::get<5>(s), std::get<6>(s),
                                   at<const int>(frames), at<const int>(positions), at<const float>(scores),
                                   at<float>(out_scores), at<int>(parents), at<int>(words), std::get<0>(n),
                                   std::get<1>(n), std::get<2>(n), std::get<3>(n), std::get<4>(n), width,
                                   beyond.flags(), at<void>(ws), ws_bytes));
          return beyond.wait();
        },
        "scores"_a, "frames"_a, "positions"_a, "beam_scores"_a, "out_scores"_a, "parents"_a, "words"_a, "sizes"_a,
        "width"_a, "validate"_a, "workspace"_a, "workspace_bytes"_a);
  // `states`: of each tensor from, to, their strides in bytes by utterance and by hypothesis, bytes of a row
  m.def("reorder_states",
        [](const std::vector<long long>& states, addr parents, int B, int N, int W, bool kept, bool validate) {
          Beyond beyond(validate);
          std::vector<tb200_states> all;
          for (size_t i = 0; i + 7 <= states.size(); i += 7) {
            const long long* s = &states[i];
            all.push_back(tb200_states{at<const void>((addr)s[0]), at<void>((addr)s[1]), s[2], s[3], s[4], s[5], s[6]});
          }
          check(tb200_reorder_states(all.data(), (int)all.size(), at<const int>(parents), B, N, W, kept,
                                     beyond.flags()));
          return beyond.wait();
        },
        "states"_a, "parents"_a, "batch_size"_a, "hypotheses"_a, "width"_a, "kept"_a, "validate"_a);
  m.def("embed_words",
        [](addr table, bool bf16, long long stride, addr words, long long count, addr rows, int R, int H, double scale,
           double dropout, long long seed, addr seed_at, bool validate) {
          Beyond beyond(validate);
          check(tb200_embed_words(at<const void>(table), bf16, stride, at<const int>(words), count, at<void>(rows), R, H,
                                  scale, dropout, seed, at<const long long>(seed_at), beyond.flags()));
          return beyond.wait();
        },
        "table"_a, "bf16"_a, "stride"_a, "words"_a, "count"_a, "rows"_a, "R"_a, "H"_a, "scale"_a, "dropout"_a, "seed"_a,
        "seed_at"_a, "validate"_a);
  m.def("embed_backward_workspace_bytes", &tb200_embed_backward_workspace_bytes);
  m.def("embed_backward",
        [](addr deltas, bool bf16, addr words, long long count, addr grad, int R, int H, double scale, double dropout,
           long long seed, addr seed_at, addr ws, size_t ws_bytes) {
          check(tb200_embed_backward(at<const void>(deltas), bf16, at<const int>(words), count, at<void>(grad), R, H,
                                     scale, dropout, seed, at<const long long>(seed_at), at<void>(ws), ws_bytes));
        },
        "deltas"_a, "bf16"_a, "words"_a, "count"_a, "grad"_a, "R"_a, "H"_a, "scale"_a, "dropout"_a, "seed"_a,
        "seed_at"_a, "workspace"_a, "workspace_bytes"_a);

  // ---- device status (bounded waits that ran out) -----------------------------------
  // Returns the code of tb200_check_status (0, or 5 = a kernel gave up) without throwing, so the
  // Python layer can raise its own exception type; the text is in last_error().
  m.def("check_status", []() { return waiting([] { return tb200_check_status(); }); });
  // (code as check_status, longest input length, longest label length), after one synchronisation;
  // the status word is left for check_status to clear
  m.def("call_summary",
        [](addr ilen, addr llen, int B, bool withStatus, addr scratch) {
          int maxLens[2] = {0, 0};
          const int rc = waiting([&] {
            return tb200_call_summary(at<const int>(ilen), at<const int>(llen), B, withStatus ? 2 : 0,
                                      at<void>(scratch), maxLens);
          });
          return py::make_tuple(rc, maxLens[0], maxLens[1]);
        },
        "input_lengths"_a, "label_lengths"_a, "batch_size"_a, "with_status"_a, "scratch"_a);
  m.def("last_error", []() { return std::string(tb200_last_error()); });
  m.def("status_name", [](int code) { return std::string(tb200_status_name(code)); }, "code"_a);
  m.def("selftest_wait_timeout",
        [](unsigned us) { check(tb200_selftest_wait_timeout(us)); }, "limit_microseconds"_a);

  m.attr("__version__") = "b200-" + std::to_string(tb200_version());
}
