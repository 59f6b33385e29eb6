// The shape of a SequencesDispatch: which sequences are active, and shapes that do
// not say. Run by tests/test_node_sequences.py.
"use strict";
const assert = require("assert");
const path = require("path");
const root = path.join(__dirname, "..", "..", "parakeet.wgsl_amd");
const host = require(path.join(root, "host"));
const addon = require(path.join(root, "lib", "pk_napi.node"));

const seen = [];
addon.countedEnqueue = (op, active) => seen.push(active);
const dispatch = new host.SequencesDispatch("step", null, {}, 4, "counted");
const encode = (shape) => dispatch.encode({ record: (fn) => fn() }, undefined, shape);
for (const [shape, want] of [
  [undefined, 4], [{ batchSize: 3 }, 3], [{ sequences: 2 }, 2], [{ batchSize: 1, rows: 188 }, 1],
  [{ batchSize: 2, sequences: 2 }, 2], [{ sequences: 4, rows: 5 }, 4]]) {
  encode(shape);
  assert.strictEqual(seen.pop(), want);
}
for (const [shape, type, message] of [
  [{}, Error, "step needs batchSize or sequences in its shape"],
  [{ rows: 2 }, Error, "step needs batchSize or sequences in its shape"],
  [{ active: 2 }, Error, "step needs batchSize or sequences in its shape"],
  [{ batchSize: 2, sequences: 3 }, Error, "step has a batchSize and sequences that differ"],
  [{ sequences: 5 }, RangeError, "step active sequences must be in [1, 4]"],
  [{ sequences: 0 }, RangeError, "step active sequences must be in [1, 4]"],
  [{ batchSize: 1.5 }, RangeError, "step active sequences must be in [1, 4]"],
  [{ sequences: "2" }, RangeError, "step active sequences must be in [1, 4]"],
  [{ sequences: null }, RangeError, "step active sequences must be in [1, 4]"]])
  assert.throws(() => encode(shape), (e) => (e instanceof type && e.message.includes(message)) || assert.fail(e.message));
assert.strictEqual(seen.length, 0);
console.log("host_cpu_sequences ok");
