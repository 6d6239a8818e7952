// CPU-only checks of the text encoder's calls over a key/value cache (no GPU): which positions Gemma3.extend and
// captureStep give to tokens when calls overlap or fail. The layer stack is replaced by one that records what it is
// given; embedding rows come from a source that answers when it is told to. Prints one JSON object.
import path from "path";
import { fileURLToPath, pathToFileURL } from "url";

const here = path.dirname(fileURLToPath(import.meta.url));
const js = path.resolve(here, "..", "..", "nanosaur2-web_amd", "js");
let Gemma3, GEMMA;

// A source of embedding rows that answers when it is told to, and an encoder whose layer stack records its calls.
function setup(batch, capacity) {
  const live = new Set();
  const tensor = (arr, shape) => {
    const t = { arr: arr.slice(), shape, buf: {}, release() { live.delete(t); } };
    live.add(t);
    return t;
  };
  const gpu = {
    fromArray: tensor,
    empty: (shape) => tensor(new Float32Array(1), shape),
    write: (buf, arr) => { buf.arr = arr.slice(); },
    capture: () => ({ result: tensor(new Float32Array(1), [1]), launch() { steps.push([...step.buf.arr]); }, destroy() {} }),
  };
  const asked = [];
  const st = { rows: (name, ids) => new Promise((resolve, reject) => asked.push({
    ids: Array.from(ids, Number),
    answer: () => resolve(new Float32Array(ids.length * GEMMA.hidden)),
    fail: () => reject(new Error("no such row")),
  })) };
  const te = new Gemma3(gpu, st);
  te.layers = [];
  const ran = [];
  const steps = [];
  let step = null;
  te.extendEmbedded = (cache, x, pos, L) => {
    ran.push({ pos: Array.from(pos.arr), L, rows: x.shape[0] });
    x.release();
    return tensor(new Float32Array(1), [1]);
  };
  const cache = { batch, capacity, bits: 16, sinks: 0, layers: [], lengths: new Array(batch).fill(0), cs: [] };
  return {
    te, cache, asked, ran, live, steps,
    recorded: () => {
      const made = new Set(live);
      const s = te.captureStep(cache);
      step = [...live].find((t) => !made.has(t) && t.arr instanceof Int32Array);
      return s;
    },
  };
}

const tick = () => new Promise((r) => setTimeout(r, 0));
// what a list of promises ends with: "ok" or the message
const ends = (ps) => Promise.all(ps.map((p) => p.then(() => "ok", (e) => String(e.message))));

async function main() {
  ({ Gemma3, GEMMA } = await import(pathToFileURL(path.join(js, "gemma3.js")).href));
  const out = {};

  {
    // two calls in flight, whose embedding rows arrive in the other order
    const s = setup(1, 16);
    const calls = [s.te.extend(s.cache, [5, 6, 7]), s.te.extend(s.cache, [8, 9])];
    const done = ends(calls);
    await tick();
    for (const a of [...s.asked].reverse()) { a.answer(); await tick(); }
    while (s.ran.length < 2 && s.asked.length) { s.asked.forEach((a) => a.answer()); await tick(); }
    out.overlap = { ends: await done, ran: [...s.ran], lengths: [...s.cache.lengths], asked: s.asked.map((a) => a.ids) };
  }
  {
    // two sequences of unequal pieces, two calls in flight
    const s = setup(2, 16);
    const calls = [s.te.extend(s.cache, [[1, 2, 3], [4]]), s.te.extend(s.cache, [[], [5, 6]])];
    const done = ends(calls);
    for (let i = 0; i < 4; i++) { s.asked.forEach((a) => a.answer()); await tick(); }
    out.batch = { ends: await done, ran: [...s.ran], lengths: [...s.cache.lengths] };
  }
  {
    // two calls that fit one by one but not together; the one that fails leaves the other alone
    const s = setup(1, 4);
    const calls = [s.te.extend(s.cache, [1, 2, 3]), s.te.extend(s.cache, [4, 5]), s.te.extend(s.cache, [6])];
    const done = ends(calls);
    for (let i = 0; i < 6; i++) { s.asked.forEach((a) => a.answer()); await tick(); }
    out.capacity = { ends: await done, ran: [...s.ran], lengths: [...s.cache.lengths] };
  }
  {
    // rows that cannot be read fail their own call only
    const s = setup(1, 8);
    const calls = [s.te.extend(s.cache, [1, 2]), s.te.extend(s.cache, [3])];
    const done = ends(calls);
    await tick();
    s.asked[0].fail();
    for (let i = 0; i < 4; i++) { s.asked.slice(1).forEach((a) => a.answer()); await tick(); }
    out.rows = { ends: await done, ran: [...s.ran], lengths: [...s.cache.lengths] };
  }
  {
    // the first call's rows come last, the second's not at all
    const s = setup(1, 8);
    const calls = [s.te.extend(s.cache, [1, 2]), s.te.extend(s.cache, [3]), s.te.extend(s.cache, [4])];
    const done = ends(calls);
    await tick();
    s.asked[1].fail();
    await tick();
    s.asked[2].answer();
    await tick();
    s.asked[0].answer();
    out.late = { ends: await done, ran: [...s.ran], lengths: [...s.cache.lengths] };
  }
  {
    // a recorded step launched, and a length set back, while rows are on their way
    const s = setup(1, 8);
    s.cache.lengths[0] = 2;
    const step = s.recorded();
    const done = ends([s.te.extend(s.cache, [1, 2])]);
    await tick();
    step.launch();
    s.asked.forEach((a) => a.answer());
    out.step = { ends: await done, ran: [...s.ran], steps: s.steps, lengths: [...s.cache.lengths] };
    const doneAgain = ends([s.te.extend(s.cache, [3])]);
    await tick();
    s.cache.lengths[0] = 1;
    s.asked.forEach((a) => a.answer());
    out.cut = { ends: await doneAgain, ran: s.ran.slice(1), lengths: [...s.cache.lengths] };
  }
  {
    // token ids as typed arrays, in a list or by themselves
    const s = setup(1, 16);
    const done = ends([s.te.extend(s.cache, [Int32Array.of(5, 6, 7)]), s.te.extend(s.cache, Uint16Array.of(8, 9)), s.te.extend(s.cache, [[1]])]);
    s.asked.forEach((a) => a.answer());
    out.typed = { ends: await done, ran: s.ran.map((r) => r.pos), asked: s.asked.map((a) => a.ids) };
  }
  {
    // the whole layer stack on a device that launches nothing, once for every launch that may fail: which tensors it
    // keeps, but for those of the op that failed
    const bf16 = (N, K) => ({ kind: "bf16", buf: { ptr: 1n }, N, K, name: "w" });
    const i4 = (N, K) => ({ ...bf16(N, K), kind: "i4", scale: { ptr: 1n }, group: 32 });
    out.failures = {};
    for (const [kind, W] of [["bf16", bf16], ["i4", i4]]) {
      const kept = [];
      let launches = Infinity;
      for (let n = 0; n <= launches && n < 100; n++) {
        const live = new Map();
        let made = 0;
        let runs = 0;
        let since = 0; // tensors made before the op that fails
        const empty = (shape, dtype = "f32") => {
          const t = { shape, dtype, buf: { ptr: 1n }, get size() { return shape.reduce((a, b) => a * b, 1); }, release() { live.delete(t); } };
          live.set(t, made++);
          return t;
        };
        const gpu = { empty, fromArray: (arr, shape) => empty(shape), run(name) {
          if (runs++ === n) throw new Error("a launch failed");
          if (name !== "te.proj" && name !== "te.mlp") since = made; // (these are the first of an op's two launches)
        } };
        const te = new Gemma3(gpu, { rows: async (name, ids) => new Float32Array(ids.length * GEMMA.hidden) });
        const norms = { inNorm: bf16(1, 1), postAttnNorm: bf16(1, 1), preMlpNorm: bf16(1, 1), postMlpNorm: bf16(1, 1), qn: bf16(1, 1), kn: bf16(1, 1) };
        const layer = (i) => ({ ...norms, global: i === 1, qkv: W(1536, 640), o: W(640, 1024), gateUp: W(4096, 640), down: W(640, 2048) });
        te.layers = [layer(0), layer(1)];
        te.norm = bf16(1, 1);
        const kv = { batch: 1, KH: 1, D: 256, capacity: 8, ldkv: 256, kvBatch: 2048 };
        const cache = { batch: 1, capacity: 8, sinks: 0, layers: [kv, kv], lengths: [0], cs: [null, null] };
        const end = (await ends([te.extend(cache, [1, 2])]))[0];
        if (end === "ok") launches = n; // every launch has failed once
        const stay = [...live.values()].filter((at) => end === "ok" || at < since).length;
        kept.push([end, stay, cache.lengths[0]]);
      }
      out.failures[kind] = kept;
    }
  }
  process.stdout.write(JSON.stringify(out) + "\n");
}

main().catch((e) => {
  process.stderr.write(`${e.stack}\n`);
  process.exit(1);
});
