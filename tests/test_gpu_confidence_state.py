"""When a decoder state has logits to score: after its own step, not after a
prefill or a batched step, and the error says which."""
import pytest

import bind as B
import voxcuda as V

pytestmark = pytest.mark.gpu


def test_a_batched_step_leaves_no_logits_and_says_so():
    V.init()
    w = B.DecoderWeights(seed=5, n_layers=1, distinct=1, vocab=8192)
    dec = V.Decoder(w.tok_emb, w.norm, [tuple(w.layer_w[0]) + tuple(w.layer_n[0])], ada_scale=w.ada_scale, vocab=w.vocab)
    states = [dec.state(kv_cap=16) for _ in range(2)]
    for st in states:
        st.prefill(B.normal_f32((4, B.DEC_DIM), 6))
        with pytest.raises(V.VoxCudaError, match="no decode step of this state alone.*prefill"):
            st.token_logprobs(0)
    tok, _ = states[0].step(B.normal_f32(B.DEC_DIM, 7))
    assert states[0].token_logprobs(tok, 1)[2].tolist() == [tok]
    V.step_batch(states, B.normal_f32((2, B.DEC_DIM), 8))
    for st in states:
        with pytest.raises(V.VoxCudaError, match="batched step"):
            st.token_logprobs(0)
        with pytest.raises(V.VoxCudaError, match="batched step"):
            st.fill_alts(2, 0.5)
    tok, _ = states[1].step(B.normal_f32(B.DEC_DIM, 9))
    assert states[1].token_logprobs(tok, 1)[2].tolist() == [tok]
    for st in states:
        st.free()
    dec.free()
