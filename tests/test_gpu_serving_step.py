"""A step of many requests through the library's operators, as a serving loop runs them:
projection with each request's adapter, normalized heads into the paged cache, attention,
output projection with adapters, log probabilities and sampling."""
import pytest
import torch

from evo_hip import native as N
import adapter_util
import test_gpu_logprobs
import test_gpu_paged_normed as normed
from adapter_util import Pool, adapt
from paged_util import CODES, DEVICE, Paged, attend, check_attention

pytestmark = pytest.mark.gpu
WIDTH, DIM, HEADS, KV, VOCAB, EPS = 256, 64, 4, 2, 512, 1e-6


class Step:
    """Weights, adapters and a batch of ragged prompts; buffers that calls in a graph keep."""

    def __init__(self, sequences, seed=0):
        self.p = Paged(sequences, heads=HEADS, kv_heads=KV, dim=DIM, seed=seed)
        self.rows = self.p.tokens
        qkv = (HEADS + 2 * KV) * DIM
        self.into = Pool(5, 16, WIDTH, qkv, ranks=[16, 8, 3, 0, 12], seed=seed)
        self.back = Pool(5, 8, HEADS * DIM, WIDTH, seed=seed + 1)
        normal = self.p.normal
        self.w_in, self.w_out, self.w_head = (
            normal(n, k, std=k ** -0.5, kind=torch.bfloat16)
            for n, k in ((qkv, WIDTH), (WIDTH, HEADS * DIM), (VOCAB, WIDTH)))
        self.scales = [1 + normal(1, DIM, std=0.2, kind=torch.float32) for _ in range(2)]
        self.inv_freq = normed.frequencies(DIM)
        self.uniform = torch.rand(self.rows, generator=self.p.gen, device=DEVICE)
        self.set_inputs(sequences)

        def empty(*shape, kind=torch.float32):
            return torch.zeros(*shape, dtype=kind, device=DEVICE)
        self.hi, self.lo = (empty(self.rows, WIDTH, kind=torch.bfloat16) for _ in range(2))
        self.shared, self.projected = empty(self.rows, qkv), empty(self.rows, qkv)
        self.query, self.out = (empty(self.rows, HEADS * DIM, kind=self.p.kind) for _ in range(2))
        self.shared_back, self.stream_out = empty(self.rows, WIDTH), empty(self.rows, WIDTH)
        self.hi2, self.lo2 = (empty(self.rows, WIDTH, kind=torch.bfloat16) for _ in range(2))
        self.logits = empty(self.rows, VOCAB)
        self.found = {n: empty(self.rows) for n in ("logprob", "entropy")}
        self.found["rank"] = empty(self.rows, kind=torch.int32)
        self.found["top_tokens"] = empty(self.rows, 4, kind=torch.int32)
        self.found["top_logprobs"] = empty(self.rows, 4)
        self.sampled = empty(self.rows, kind=torch.int32)
        need = max(N.call("evo_hip_adapter_linear_workspace_bytes", pool.struct(), self.rows)
                   for pool in (self.into, self.back))
        self.adapters_space = torch.zeros(need, dtype=torch.uint8, device=DEVICE)
        need = N.call("evo_hip_paged_attention_workspace_bytes", self.p.cache(), self.p.batch(),
                      HEADS)
        self.attention_space = torch.zeros(max(need, 16), dtype=torch.uint8, device=DEVICE)

    def set_inputs(self, sequences):
        """Each sequence's rows have one adapter, or none."""
        self.x = self.p.normal(self.rows, WIDTH, kind=torch.float32)
        ids = []
        for n, _ in sequences:
            ids += [int(torch.randint(-1, 5, (1,), generator=self.p.gen, device=DEVICE))] * n
        self.of_rows = self.p.ints(ids)
        self.tokens = torch.randint(0, VOCAB, (self.rows,), generator=self.p.gen,
                                    device=DEVICE).to(torch.int32)

    def linear(self, hi, lo, w, out, stream):
        N.call("evo_hip_linear", hi.data_ptr(), None if lo is None else lo.data_ptr(),
               w.data_ptr(), None, None, hi.shape[0], w.shape[0], w.shape[1], out.data_ptr(),
               stream.cuda_stream)

    def run(self, stream=None):
        s = torch.cuda.current_stream() if stream is None else stream
        p = self.p
        N.call("evo_hip_split_f32", self.x.data_ptr(), self.x.numel(), self.hi.data_ptr(),
               self.lo.data_ptr(), s.cuda_stream)
        self.linear(self.hi, self.lo, self.w_in, self.shared, s)
        adapt(self.into, self.of_rows, self.hi, self.lo, self.shared, self.projected, s,
              self.adapters_space)
        N.call("evo_hip_paged_append_normed", p.cache(), p.batch(), N.DTYPE_F32,
               self.projected.data_ptr(), self.projected.stride(0), HEADS, 0,
               self.scales[0].data_ptr(), self.scales[1].data_ptr(), 0, EPS, 1,
               self.inv_freq.data_ptr(), DIM, 0, 1.0, self.query.data_ptr(),
               self.query.stride(0), s.cuda_stream)
        attend(p, self.query, DIM ** -0.5, out=self.out, stream=s, workspace=self.attention_space)
        self.linear(self.out, None, self.w_out, self.shared_back, s)
        adapt(self.back, self.of_rows, self.out, None, self.shared_back, self.stream_out, s,
              self.adapters_space)
        N.call("evo_hip_split_f32", self.stream_out.data_ptr(), self.stream_out.numel(),
               self.hi2.data_ptr(), self.lo2.data_ptr(), s.cuda_stream)
        self.linear(self.hi2, self.lo2, self.w_head, self.logits, s)
        f = self.found
        N.call("evo_hip_token_logprobs", N.DTYPE_F32, self.logits.data_ptr(), self.rows, VOCAB,
               VOCAB, self.tokens.data_ptr(), f["logprob"].data_ptr(), f["rank"].data_ptr(),
               f["entropy"].data_ptr(), 4, f["top_tokens"].data_ptr(),
               f["top_logprobs"].data_ptr(), None, 0, s.cuda_stream)
        N.call("evo_hip_sample", N.DTYPE_F32, self.logits.data_ptr(), self.rows, VOCAB, VOCAB,
               None, None, None, None, self.uniform.data_ptr(), self.sampled.data_ptr(), None, 0,
               s.cuda_stream)

    def results(self):
        return [self.projected, self.query, self.p.keys.nan_to_num(), self.p.values.nan_to_num(),
                self.out, self.stream_out, self.logits, *self.found.values(), self.sampled]

    def check(self):
        """Each operator against its definition, on what it was given."""
        p = self.p
        adapter_util.check(self.into, self.of_rows, self.hi, self.lo, self.shared, self.projected)
        x = self.projected.view(self.rows, HEADS + 2 * KV, DIM)
        position = torch.tensor([q for _, _, q in p.rows()], device=DEVICE)
        page = torch.tensor([p.page_of(s, q) for _, s, q in p.rows()], device=DEVICE)
        slot = position % p.page
        for got, source, weight in (
                (self.query.view(self.rows, HEADS, DIM), x[:, :HEADS], self.scales[0]),
                (p.keys[page, :, slot], x[:, HEADS:HEADS + KV], self.scales[1])):
            expected, far = normed.exact_heads(source, weight, EPS, True, position, DIM, False, 1.0)
            normed.within(got, expected, far, p.kind)
        assert torch.equal(p.values[page, :, slot], x[:, HEADS + KV:].to(p.kind))
        check_attention(p, self.query, DIM ** -0.5, self.out)
        adapter_util.check(self.back, self.of_rows, self.out, None, self.shared_back,
                           self.stream_out)
        test_gpu_logprobs.check(self.logits, self.tokens, 4, self.found)
        assert p.error.item() == 0 and self.into.error.item() == 0


def test_prompts_and_a_decode_step_together():
    """Prompts of ragged lengths beside requests that add one token, every operator checked."""
    step = Step([(37, 37), (1, 1), (90, 90), (1, 1), (16, 16)])
    step.run()
    step.check()


def test_captured_steps_follow_their_inputs():
    """A decode step in one graph: new tokens, adapters and lengths, replays beside eager
    work, each equal to the eager step bit for bit."""
    sequences = [(1, 60 + 7 * i) for i in range(20)]
    step = Step(sequences, seed=3)
    lengths = [20 + i for i in range(20)]
    # (Positions in front of the first step's hold what some earlier step appended.)
    for pool in (step.p.keys, step.p.values):
        pool.copy_(step.p.normal(*pool.shape))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step.p.lengths.copy_(step.p.ints(lengths))
        step.run(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    x, of_rows, tokens = step.x, step.of_rows, step.tokens
    with torch.cuda.graph(graph, stream=side):
        step.run(side)
    for i in range(1, 6):
        step.p.lengths.copy_(step.p.ints([n + i for n in lengths]))
        step.set_inputs(sequences)
        x.copy_(step.x)
        of_rows.copy_(step.of_rows)
        tokens.copy_(step.tokens)
        step.x, step.of_rows, step.tokens = x, of_rows, tokens
        keys, values = step.p.keys.clone(), step.p.values.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [r.clone() for r in step.results()]
        step.p.keys.copy_(keys)
        step.p.values.copy_(values)
        step.run()
        torch.cuda.synchronize()
        for a, b in zip(replayed, step.results()):
            assert torch.equal(a, b)
    assert CODES[step.p.kind] == N.DTYPE_BF16 and step.p.error.item() == 0
