"""Continuous batching over a LanguageModel: requests wait for a slot, prompts are taken in portions that share steps
with the sequences already decoding, and when no prompt is left to read the running sequences decode together on the
device (one graph replay per token) until one of them is due to end.  Sampling is greedy, on the device.

generate_drafted samples at a temperature, with a second model that proposes tokens."""
from collections import deque


def pages_to_come(model, slot, most):
    """Pages that a slot has still to take until it holds `most`."""
    return most - -(-model.length[slot] // model.page)


class Request:
    def __init__(self, prompt, max_new, stop=()):
        self.prompt, self.max_new, self.stop = [int(t) for t in prompt], int(max_new), frozenset(stop)
        self.slot, self.done, self.output = None, 0, []  # done: prompt tokens read so far

    @property
    def finished(self):
        return len(self.output) >= self.max_new or bool(self.output and self.output[-1] in self.stop)


class Scheduler:
    def __init__(self, model, portion=None, stop_check=16):
        """portion: most prompt tokens of one request in a step (default: the model's max_rows); stop_check: decode
        steps between looks at the stop tokens."""
        self.model, self.portion, self.stop_check = model, portion or model.max_rows, stop_check
        self.waiting, self.running = deque(), []
        self.page, self.pages = getattr(model, "page", 0), getattr(model, "pages", 0)

    def _pages(self, r):
        """Pages that a request holds at most."""
        return (len(r.prompt) + r.max_new + self.page - 1) // self.page if self.page else 0

    def _room(self, r):
        """Whether a request finds its pages beside what those that run have still to take, whoever else holds some."""
        return not self.page or sum(pages_to_come(self.model, x.slot, self._pages(x)) for x in self.running) + self._pages(r) <= self.model.free_pages()

    def submit(self, prompt, max_new, stop=()):
        r = Request(prompt, max_new, stop)
        if not r.prompt or r.max_new < 1:
            raise ValueError("a request needs a prompt and at least one new token")
        if len(r.prompt) + r.max_new > self.model.max_ctx:
            raise ValueError(f"{len(r.prompt)} + {r.max_new} tokens do not fit a slot of {self.model.max_ctx}")
        if self._pages(r) > self.pages:
            raise ValueError(f"{len(r.prompt)} + {r.max_new} tokens do not fit {self.pages} pages of {self.page}")
        self.waiting.append(r)
        return r

    def _admit(self):
        while self.waiting:
            if not self._room(self.waiting[0]):
                return
            slot = self.model.acquire()
            if slot is None:
                return
            r = self.waiting.popleft()
            r.slot = slot
            self.running.append(r)

    def _retire(self):
        for r in [r for r in self.running if r.finished]:
            self.running.remove(r)
            self.model.release(r.slot)

    def _mixed_step(self):
        m = self.model
        room, entries, ends = m.max_rows, [], []
        for r in self.running:  # sequences that decode come first, a token each
            if r.done == len(r.prompt) and room:
                entries.append((r.slot, [r.output[-1]]))
                ends.append(r)
                room -= 1
        for r in self.running:
            n = min(len(r.prompt) - r.done, self.portion, room)
            if n > 0:
                entries.append((r.slot, r.prompt[r.done:r.done + n]))
                r.done += n
                room -= n
                if r.done == len(r.prompt):
                    ends.append(r)
        m.step(entries, sample=True)
        for r in ends:
            r.output.append(int(m.read(r.slot, m.length[r.slot] - 1, 1)[0]))

    def _decode(self):
        m = self.model
        steps = min(r.max_new - len(r.output) for r in self.running)
        if any(r.stop for r in self.running):
            steps = min(steps, self.stop_check)
        batch = self.running[:m.max_rows]
        first = {r.slot: m.length[r.slot] for r in batch}
        m.decode([r.slot for r in batch], steps)
        for r in batch:
            for t in m.read(r.slot, first[r.slot], steps):
                if not r.finished:
                    r.output.append(int(t))

    def run(self):
        """Until every submitted request is finished."""
        while self.waiting or self.running:
            self._admit()
            if not self.running:
                raise RuntimeError("no slot or too few pages for a request: others hold them")
            if any(r.done < len(r.prompt) for r in self.running):
                self._mixed_step()
            else:
                self._decode()
            self._retire()


class _Drafted:
    def __init__(self, prompt, max_new, stop, slots):
        self.tokens, self.start, self.end, self.stop = [int(t) for t in prompt], len(prompt), len(prompt) + int(max_new), frozenset(stop)
        self.slot, self.draft_slot = slots

    @property
    def finished(self):
        return len(self.tokens) >= self.end or (len(self.tokens) > self.start and self.tokens[-1] in self.stop)


def generate_drafted(model, draft, prompts, max_new, drafts=4, temperature=0.0, seed=0, stop=(), portion=None):
    """Continuations of all prompts: `draft`, a smaller model of the same vocabulary, proposes `drafts` tokens a round, `model`
    looks at all of them in one step, and what stands is decided so that the tokens are draws of `model` at this temperature (0:
    its greedy tokens).  Both models' sequences are taken back to what stood, so neither may have layers that cannot go back."""
    import torch

    from . import drafts as ops
    from . import lm
    for m in (model, draft):
        if m.config["conv_taps"] > 1 or any(d["mixer"] == lm.RETENTION for d in m.layers):
            raise ValueError("models with retention or an input convolution cannot take drafted tokens back")
    if draft.vocab != model.vocab:
        raise ValueError("the draft model has another vocabulary")
    if not 1 <= drafts <= 64 or drafts + 1 > min(model.max_rows, draft.max_rows):  # (models with windows go back by 64 tokens)
        raise ValueError(f"{drafts} drafts a round")
    waiting, running, out = deque(enumerate(prompts)), {}, [None] * len(prompts)
    for p in prompts:
        if not len(p) or max_new < 1 or len(p) + max_new > min(model.max_ctx, draft.max_ctx):
            raise ValueError("a request needs a prompt, at least one new token, and room for both in a slot of both models")
    held = lambda m, n: -(-(n + max_new) // m.page) if m.page else 0  # pages that a prompt of n tokens and what follows it take
    roles = lambda m: (m is model) + (m is draft)
    for m in (model, draft):
        if any(held(m, len(p)) * roles(m) > m.pages for p in prompts):
            raise ValueError(f"a request does not fit {m.pages} pages of {m.page}")

    def room(m, n):  # whether a prompt of n tokens finds its pages beside what the others have still to take
        to_come = lambda r: sum(pages_to_come(m, s, held(m, r.start)) for x, s in ((model, r.slot), (draft, r.draft_slot)) if x is m)
        return not m.page or sum(map(to_come, running.values())) + held(m, n) * roles(m) <= m.free_pages()

    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, generator=gen, device="cuda")

    def read(m, slot, tokens):  # tokens that nobody asks about
        n = min(portion or m.max_rows, m.max_rows)
        for i in range(0, len(tokens), n):
            m.step([(slot, tokens[i:i + n])])

    def round_of(batch):
        # as many drafts for all of the batch as the one with the least room takes; one place is the target's own token
        k = min([drafts] + [r.end - len(r.tokens) - 1 for r in batch])
        if k:
            for r in batch:  # all but the last token, which the proposals' first step reads
                read(draft, r.draft_slot, r.tokens[draft.length[r.draft_slot]:-1])
        q = torch.empty((len(batch), k, model.vocab), dtype=torch.float32, device="cuda")
        none = torch.empty((len(batch), 0, model.vocab), dtype=torch.float32, device="cuda")
        no_tokens, no_accept = none.new_empty((len(batch), 0), dtype=torch.int32), none.new_empty((len(batch), 0))
        proposed = torch.empty((len(batch), k), dtype=torch.int32, device="cuda")
        last = [r.tokens[-1] for r in batch]
        for i in range(k):
            draft.step_probabilities([(r.draft_slot, [t]) for r, t in zip(batch, last)], range(len(batch)), temperature, out=q[:, i])
            _, new = ops.verify(q[:, i:i + 1], none, no_tokens, no_accept, rand(len(batch)))
            proposed[:, i] = new[:, 0]
            last = new[:, 0].tolist()
            if min(last) < 0:
                raise RuntimeError("the draft model's probabilities have no mass")
        names = proposed.tolist()
        p = model.step_probabilities([(r.slot, [r.tokens[-1]] + x) for r, x in zip(batch, names)], range(len(batch) * (k + 1)), temperature)
        accepted, new = ops.verify(p.view(len(batch), k + 1, -1), q, proposed, rand(len(batch), k), rand(len(batch)))
        for r, n, x in zip(batch, accepted.tolist(), new.tolist()):
            if x[n] < 0:
                raise RuntimeError("the model's probabilities have no mass")
            stand = len(r.tokens) + n  # tokens that both models may keep
            model.truncate(r.slot, min(model.length[r.slot], stand))
            if k:
                draft.truncate(r.draft_slot, min(draft.length[r.draft_slot], stand))
            for t in x[:n + 1]:
                if not r.finished:
                    r.tokens.append(t)

    try:
        while waiting or running:
            while waiting:
                if not all(room(m, len(waiting[0][1])) for m in (model, draft)):
                    break
                slots = model.acquire(), draft.acquire()
                if None in slots:
                    for m, s in zip((model, draft), slots):
                        if s is not None:
                            m.release(s)
                    break
                i, p = waiting.popleft()
                running[i] = _Drafted(p, max_new, stop, slots)
                read(model, slots[0], running[i].tokens[:-1])
            if not running:
                raise RuntimeError("no slot or too few pages for a request: others hold them")
            batch = list(running.values())
            most = max(1, min(model.max_rows // (drafts + 1), draft.max_rows))
            for b in range(0, len(batch), most):
                round_of(batch[b:b + most])
            for i in [i for i, r in running.items() if r.finished]:
                r = running.pop(i)
                out[i] = r.tokens[r.start:]
                model.release(r.slot)
                draft.release(r.draft_slot)
    except BaseException:
        for r in running.values():
            model.release(r.slot)
            draft.release(r.draft_slot)
        raise
    return out


def generate(model, prompts, max_new, stop=(), portion=None):
    """Greedy continuations of all prompts, batched."""
    s = Scheduler(model, portion)
    reqs = [s.submit(p, max_new, stop) for p in prompts]
    s.run()
    return [r.output for r in reqs]
